// host_logits.cpp - the host side of logit adjustment and the LM head (fsb_logits.cpp) over the same stand-in for the device as
// host_order.cpp: what is refused, what the kernels are told, and what a call that fails leaves behind.  Prints "ok", or what went wrong.
#define main host_order_main
#include "host_order.cpp"
#undef main

#include <array>
#include <cmath>
#include <memory>

namespace {
struct Seen {            // an adjustment as it was queued, and the window and biases that it read when its turn came
    fsb::AdjustArgs a;
    std::vector<fsb::AdjustRow> rows;
    std::vector<std::vector<int32_t>> windows, biases;
};
std::vector<std::shared_ptr<Seen>> adjusted_;
std::vector<fsb::HeadArgs> heads_;
int empty_row_ = -1;     // the next adjustment reports this row
bool late_ = false;      // the next head launch gives up
}  // namespace

extern "C" cudaError_t cudaDeviceSynchronize() { run_until(nullptr); return cudaSuccess; }

namespace fsb {
int launch_adjust(const AdjustArgs& a, const AdjustRow* rows, void*, int* launches) {
    auto s = std::make_shared<Seen>();
    s->a = a;
    s->rows.assign(rows, rows + a.n_rows);
    adjusted_.push_back(s);
    const int empty = empty_row_;
    empty_row_ = -1;
    enqueue([=] {
        for (const AdjustRow& r : s->rows) {
            s->windows.emplace_back(a.pool + r.hist_begin, a.pool + r.hist_begin + r.hist_len);
            s->biases.emplace_back(a.pool + r.bias_begin, a.pool + r.bias_begin + 2 * r.n_bias);
        }
        if (empty >= 0 && a.row_state) *a.empty = 1u + (uint32_t)empty;
    });
    ++*launches;
    return 0;
}
int64_t head_weight_bytes(int v, int k) { return (int64_t)v * k; }
int64_t head_scale_bytes(int v, int k, int) { return (int64_t)v * k; }
int launch_head_layout(const unsigned char*, const void*, int, int, int, unsigned char*, unsigned char*, void*) { return 0; }
int prepare_head_kernels() { return 0; }
int launch_head(const HeadArgs& a, void*, int* launches) {
    heads_.push_back(a);
    const bool late = late_;
    late_ = false;
    enqueue([=] {
        if (late) *a.late = 1u;
    });
    ++*launches;
    return 0;
}
}  // namespace fsb

namespace {
alignas(16) float rows_[4000], out_[4000];
alignas(16) uint8_t weights_[1000 * 32];
alignas(16) uint16_t scales_[1000 * 2], hidden_[8 * 64];
uint32_t masks_[4 * 32];

#define WANT(what, call, code)                                         \
    do {                                                               \
        const long long got_ = (call);                                 \
        if (got_ != (code)) return bad(what, __LINE__, got_, (code));  \
    } while (0)

int adjust(Setup& s, int n) {
    return fsb_adjust_logits(s.h, n, s.sid.data(), rows_, FSB_F32, 1000, 1000, nullptr, 0, 0, nullptr, out_, FSB_F32, 1000);
}

// What an adjustment is told about its rows, and that nothing of a closed stream is left for the next one.
int settings() {
    Setup s(2, 1.0f);
    const int32_t hist[6] = {5, 6, 7, 7, 8, 9}, ids[3] = {30, 10, 20};
    const float values[3] = {3.0f, 1.0f, -INFINITY};
    fsb_stream_history_set(s.h, s.sid[0], hist, 6);
    WANT("penalties", fsb_stream_penalties_set(s.h, s.sid[0], 0.5f, 0.25f), FSB_OK);
    WANT("bias", fsb_stream_bias_set(s.h, s.sid[0], ids, values, 3), FSB_OK);
    WANT("adjust", adjust(s, 2), FSB_OK);
    run_until(nullptr);
    const Seen& a = *adjusted_.back();
    if (a.windows[0] != std::vector<int32_t>(hist, hist + 6)) return bad("window", 0, (long long)a.windows[0].size(), 6);
    if (a.rows[0].frequency != 0.5f || a.rows[0].presence != 0.25f || a.rows[0].repetition != 1.0f) return bad("penalties", 1, 0, 1);
    if (a.biases[0].size() != 6 || a.biases[0][0] != 10 || a.biases[0][1] != 20 || a.biases[0][2] != 30) return bad("bias ids", 0, (long long)a.biases[0].size(), 6);
    float v[3];
    std::memcpy(v, &a.biases[0][3], sizeof v);
    if (v[0] != 1.0f || v[1] != -INFINITY || v[2] != 3.0f) return bad("bias values", 0, 0, 1);
    if (a.rows[1].hist_len != 0 || a.rows[1].n_bias != 0 || a.rows[1].mask_row != -1) return bad("other row", 0, 1, 0);
    // the id is used again
    fsb_stream_close(s.h, s.sid[0]);
    ferro_sampler_params p;
    fsb_params_default(&p);
    p.repetition_penalty = 1.0f;
    p.seed = 1;
    int again = -1;
    fsb_stream_open(s.h, &p, &again);
    if (again != s.sid[0]) return bad("id", 0, again, s.sid[0]);
    fsb_stream_history_set(s.h, again, hist, 6);
    WANT("adjust", adjust(s, 2), FSB_OK);
    const fsb::AdjustRow& r = adjusted_.back()->rows[0];
    if (r.n_bias != 0 || r.frequency != 0.0f || r.presence != 0.0f || r.hist_len != 0) return bad("settings of a closed stream", 0, r.n_bias, 0);
    // windows: cut by repeat_last_n and penalty_from, whatever the repetition penalty
    for (const auto& c : {std::array<int, 3>{-1, 0, 6}, {2, 0, 2}, {0, 0, 0}, {-1, 4, 2}, {5, 4, 2}, {100, 0, 6}, {-1, 9, 0}}) {
        fsb_stream_close(s.h, s.sid[0]);
        p.repeat_last_n = c[0];
        p.penalty_from = c[1];
        fsb_stream_open(s.h, &p, &again);
        fsb_stream_history_set(s.h, again, hist, 6);
        fsb_stream_penalties_set(s.h, again, 1.0f, 0.0f);
        WANT("adjust", adjust(s, 1), FSB_OK);
        run_until(nullptr);
        if (adjusted_.back()->windows[0] != std::vector<int32_t>(hist + 6 - c[2], hist + 6)) return bad("window", c[0] * 100 + c[1], (long long)adjusted_.back()->windows[0].size(), c[2]);
    }
    return 0;
}

// Regions of the id pool: lists that grow and shrink, a list that finds no room, many streams one after the other.
int regions() {
    fsb_handle* h = nullptr;
    fsb_create(0, 2, 1000, 1024, &h);      // four regions of the smallest size
    ferro_sampler_params p;
    fsb_params_default(&p);
    p.seed = 1;
    std::vector<int32_t> ids(600);
    std::vector<float> v(600, 1.0f);
    for (int i = 0; i < 600; ++i) ids[(size_t)i] = 600 - i;
    for (int k = 0; k < 50; ++k) {
        int sid = 0;
        fsb_stream_open(h, &p, &sid);
        WANT("small", fsb_stream_bias_set(h, sid, ids.data(), v.data(), 5), FSB_OK);
        WANT("larger", fsb_stream_bias_set(h, sid, ids.data(), v.data(), 200), FSB_OK);
        WANT("too large", fsb_stream_bias_set(h, sid, ids.data(), v.data(), 600), FSB_ERR_CAPACITY);
        WANT("adjust", fsb_adjust_logits(h, 1, &sid, rows_, FSB_F32, 1000, 1000, nullptr, 0, 0, nullptr, out_, FSB_F32, 1000), FSB_OK);
        if (adjusted_.back()->rows[0].n_bias != 200) return bad("biases after a refused list", k, adjusted_.back()->rows[0].n_bias, 200);
        WANT("none", fsb_stream_bias_set(h, sid, nullptr, nullptr, 0), FSB_OK);
        WANT("close", fsb_stream_close(h, sid), FSB_OK);
    }
    fsb_destroy(h);
    return 0;
}

// Sampling adjusted rows: never ahead of the kernel that writes them, and a call that fails leaves streams and histories as they were.
int sampling() {
    Setup s(3, 1.2f);
    const int32_t ids[3] = {1, 2, 3};
    for (int sid : s.sid) fsb_stream_history_set(s.h, sid, ids, 3);
    fsb_set_launch_overlap(s.h, 1);
    int32_t tok[3] = {-7, -7, -7};
    auto call = [&] {
        return fsb_sample_batch_adjusted(s.h, 3, s.sid.data(), rows_, FSB_F32, 1000, 1000, nullptr, 0, 0, nullptr, tok, FSB_APPEND_SAMPLED);
    };
    overlaps_.clear();
    for (int step = 0; step < 3; ++step) {
        // a row without a token
        uint64_t draws = 0;
        int64_t len = 0;
        empty_row_ = 1;
        std::memset(tok, 0xff, sizeof tok);
        WANT("empty", call(), FSB_ERR_EMPTY);
        if (tok[0] != -1) return bad("token of a failed call", step, tok[0], -1);
        for (int sid : s.sid) {
            fsb_stream_state_get(s.h, sid, nullptr, &draws);
            fsb_stream_history_len(s.h, sid, &len);
            if (draws != (uint64_t)step || len != 3 + step) return bad("stream after a failed call", step, (long long)draws, step);
        }
        const auto want = s.next();
        WANT("call", call(), FSB_OK);
        for (int i = 0; i < 3; ++i)
            if (tok[i] != want[(size_t)i]) return bad("token", step * 10 + i, tok[i], want[(size_t)i]);
        run_until(nullptr);
        const auto& w = adjusted_.back()->windows;   // the tokens that were appended before
        for (int i = 0; i < 3; ++i)
            if ((int)w[(size_t)i].size() != 3 + step) return bad("window", step, (long long)w[(size_t)i].size(), 3 + step);
    }
    for (int m : overlaps_)
        if (m != 2) return bad("mode of launch", 0, m, 2);
    // the engine's own mode is back
    fsb_batch* b = s.prepare();
    fsb_batch_launch(s.h, b, logits_);
    if (overlaps_.back() != 1) return bad("mode afterwards", 0, overlaps_.back(), 1);
    return 0;
}

int head() {
    Setup s(2, 1.2f);
    fsb_head* head = nullptr;
    WANT("create", fsb_head_create(s.h, 1000, 64, 32, weights_, scales_, FSB_F16, 0, &head), FSB_OK);
    const int32_t ids[3] = {1, 2, 3};
    for (int sid : s.sid) fsb_stream_history_set(s.h, sid, ids, 3);
    int32_t tok[2];
    auto call = [&](const uint32_t* masks) {
        return fsb_sample_hidden(s.h, head, 2, s.sid.data(), hidden_, FSB_BF16, 64, masks, 32, masks ? 2 : 0, nullptr, tok, FSB_APPEND_SAMPLED);
    };
    // without masks and settings: no adjustment
    const size_t before = adjusted_.size();
    auto want = s.next();
    WANT("hidden", call(nullptr), FSB_OK);
    if (tok[0] != want[0] || adjusted_.size() != before) return bad("plain step", 0, (long long)adjusted_.size(), (long long)before);
    want = s.next();
    WANT("hidden", call(masks_), FSB_OK);
    if (tok[1] != want[1] || adjusted_.size() != before + 1) return bad("masked step", 0, (long long)adjusted_.size(), (long long)before + 1);
    if (adjusted_.back()->a.in != adjusted_.back()->a.out || heads_.back().logits != adjusted_.back()->a.in) return bad("in place", 0, 0, 1);
    // a launch that gives up
    for (const uint32_t* masks : {(const uint32_t*)nullptr, (const uint32_t*)masks_}) {
        late_ = true;
        WANT("late", call(masks), FSB_ERR_DEVICE);
        uint64_t draws = 0;
        int64_t len = 0;
        fsb_stream_state_get(s.h, s.sid[0], nullptr, &draws);
        fsb_stream_history_len(s.h, s.sid[0], &len);
        if (draws != 2 || len != 5) return bad("stream after a launch that gave up", 0, (long long)draws, 2);
    }
    want = s.next();
    WANT("afterwards", call(masks_), FSB_OK);
    if (tok[0] != want[0]) return bad("token", 0, tok[0], want[0]);
    // ... that nobody waited for: the next call tells
    late_ = true;
    auto logits = [&] { return fsb_head_logits(s.h, head, 2, hidden_, FSB_BF16, 64, out_, 1000); };
    WANT("queued", logits(), FSB_OK);
    run_until(nullptr);
    WANT("told", logits(), FSB_ERR_DEVICE);
    WANT("again", logits(), FSB_OK);
    // memory that two captured launches would share is not handed to them
    if (heads_.back().scratch_rows != 2 || !heads_.back().chained) return bad("eager launch", 0, heads_.back().scratch_rows, 2);
    capturing_ = true;
    const int rc = logits();
    capturing_ = false;
    WANT("captured", rc, FSB_OK);
    if (heads_.back().scratch_rows != 0 || heads_.back().chained) return bad("captured launch", 0, heads_.back().scratch_rows, 0);
    Setup other(1);
    WANT("another engine's", fsb_head_free(other.h, head), FSB_ERR_INVALID);
    WANT("free", fsb_head_free(s.h, head), FSB_OK);
    WANT("freed", logits(), FSB_ERR_INVALID);
    WANT("freed twice", fsb_head_free(s.h, head), FSB_ERR_INVALID);
    return 0;
}

int refusals() {
    Setup s(3, 1.1f);
    int32_t tok[4] = {};
    const int twice[2] = {s.sid[0], s.sid[0]}, unknown[2] = {s.sid[0], 99};
    auto adj = [&](int n, const int* sid, const void* lg, int type, int64_t ld, int V, const uint32_t* m, int64_t mld, int nm, const int32_t* mr, void* out, int otype, int64_t old) {
        return fsb_adjust_logits(s.h, n, sid, lg, type, ld, V, m, mld, nm, mr, out, otype, old);
    };
    const int* sid = s.sid.data();
    char* odd = reinterpret_cast<char*>(rows_) + 1;
    WANT("fine", adj(2, sid, rows_, 0, 1000, 1000, masks_, 32, 2, nullptr, out_, 0, 1000), FSB_OK);
    WANT("twice", adj(2, twice, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_OK);
    WANT("in place", adj(2, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, rows_, 0, 1000), FSB_OK);
    WANT("handle", fsb_adjust_logits(nullptr, 1, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("streams", adj(2, nullptr, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("unknown", adj(2, unknown, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_STREAM_ID);
    WANT("no rows", adj(0, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("rows", adj(4, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_CAPACITY);
    WANT("no columns", adj(1, sid, rows_, 0, 1000, 0, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("columns", adj(1, sid, rows_, 0, 1001, 1001, nullptr, 0, 0, nullptr, out_, 0, 1001), FSB_ERR_CAPACITY);
    WANT("logits", adj(1, sid, nullptr, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("out", adj(1, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, nullptr, 0, 1000), FSB_ERR_INVALID);
    WANT("stride", adj(1, sid, rows_, 0, 999, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("out stride", adj(1, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 999), FSB_ERR_INVALID);
    WANT("type", adj(1, sid, rows_, 3, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("types", adj(1, sid, rows_, 1, 1000, 1000, nullptr, 0, 0, nullptr, out_, 2, 1000), FSB_ERR_INVALID);
    WANT("fp32 to bf16", adj(1, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 1, 1000), FSB_ERR_INVALID);
    WANT("alignment", adj(1, sid, odd, 0, 1000, 900, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("alignment", adj(1, sid, odd, 1, 1000, 900, nullptr, 0, 0, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("overlap", adj(2, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, rows_ + 1, 0, 1000), FSB_ERR_INVALID);
    WANT("overlap", adj(2, sid, rows_, 0, 1000, 900, nullptr, 0, 0, nullptr, rows_, 0, 900), FSB_ERR_INVALID);
    WANT("behind", adj(2, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, rows_ + 2000, 0, 1000), FSB_OK);
    WANT("mask words", adj(2, sid, rows_, 0, 1000, 1000, masks_, 31, 2, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("masks", adj(2, sid, rows_, 0, 1000, 1000, masks_, 32, 1, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    const int32_t high[2] = {0, 2}, low[2] = {-2, 0}, some[2] = {-1, 1};
    WANT("mask row", adj(2, sid, rows_, 0, 1000, 1000, masks_, 32, 2, high, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("mask row", adj(2, sid, rows_, 0, 1000, 1000, masks_, 32, 2, low, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("mask rows", adj(2, sid, rows_, 0, 1000, 1000, masks_, 32, 2, some, out_, 0, 1000), FSB_OK);
    WANT("no masks", adj(2, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, some, out_, 0, 1000), FSB_ERR_INVALID);
    fsb_set_vocab_offset(s.h, 40);
    WANT("mask words of a shard", adj(2, sid, rows_, 0, 1000, 1000, masks_, 32, 2, nullptr, out_, 0, 1000), FSB_ERR_INVALID);
    WANT("mask words of a shard", adj(2, sid, rows_, 0, 1000, 1000, masks_, 33, 2, nullptr, out_, 0, 1000), FSB_OK);
    fsb_set_vocab_offset(s.h, 0);
    capturing_ = true;
    int rc = adj(2, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, out_, 0, 1000);
    const int32_t id = 4;
    const float one = 1.0f;
    const int rc2 = fsb_stream_bias_set(s.h, s.sid[0], &id, &one, 1);
    const int rc3 = fsb_sample_batch_adjusted(s.h, 1, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, tok, 0);
    capturing_ = false;
    WANT("captured", rc, FSB_ERR_INVALID);
    WANT("captured", rc2, FSB_ERR_INVALID);
    WANT("captured", rc3, FSB_ERR_INVALID);
    auto samp = [&](int n, const int* ids, unsigned flags) { return fsb_sample_batch_adjusted(s.h, n, ids, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, tok, flags); };
    WANT("twice", samp(2, twice, 0), FSB_ERR_INVALID);
    for (unsigned f : {(unsigned)FSB_LOGITS_ON_HOST, (unsigned)FSB_WRITE_BACK, 64u}) WANT("flags", samp(2, sid, f), FSB_ERR_INVALID);
    WANT("tokens", fsb_sample_batch_adjusted(s.h, 1, sid, rows_, 0, 1000, 1000, nullptr, 0, 0, nullptr, nullptr, 0), FSB_ERR_INVALID);
    fsb_set_vocab_shard(s.h, 0, 2000);
    WANT("shard", samp(2, sid, 0), FSB_ERR_INVALID);
    fsb_set_vocab_shard(s.h, 0, 0);
    uint64_t draws = 1;
    fsb_stream_state_get(s.h, s.sid[0], nullptr, &draws);
    WANT("draws", (long long)draws, 0);
    for (float v : {INFINITY, -INFINITY, NAN}) {
        WANT("penalty", fsb_stream_penalties_set(s.h, s.sid[0], v, 0.0f), FSB_ERR_RANGE);
        WANT("penalty", fsb_stream_penalties_set(s.h, s.sid[0], 0.0f, v), FSB_ERR_RANGE);
        WANT("bias", fsb_stream_bias_set(s.h, s.sid[0], &id, &v, 1), v == -INFINITY ? FSB_OK : FSB_ERR_RANGE);
    }
    const int32_t same[2] = {3, 3};
    const float two[2] = {1.0f, 1.0f};
    WANT("bias twice", fsb_stream_bias_set(s.h, s.sid[0], same, two, 2), FSB_ERR_INVALID);
    WANT("bias", fsb_stream_bias_set(s.h, s.sid[0], nullptr, two, 2), FSB_ERR_INVALID);
    WANT("bias", fsb_stream_bias_set(s.h, s.sid[0], same, two, -1), FSB_ERR_INVALID);
    WANT("bias", fsb_stream_bias_set(s.h, 99, same, two, 1), FSB_ERR_STREAM_ID);
    WANT("penalties", fsb_stream_penalties_set(s.h, 99, 0.0f, 0.0f), FSB_ERR_STREAM_ID);
    fsb_head* head = nullptr;
    auto create = [&](int V, int K, int g, const void* w, const void* sc, int type, unsigned flags) {
        return fsb_head_create(s.h, V, K, g, static_cast<const uint8_t*>(w), sc, type, flags, &head);
    };
    WANT("vocabulary", create(0, 64, 32, weights_, scales_, FSB_F16, 0), FSB_ERR_CAPACITY);
    WANT("vocabulary", create((1 << 20) + 1, 64, 32, weights_, scales_, FSB_F16, 0), FSB_ERR_CAPACITY);
    WANT("group", create(1000, 64, 16, weights_, scales_, FSB_F16, 0), FSB_ERR_RANGE);
    WANT("hidden", create(1000, 96, 64, weights_, scales_, FSB_F16, 0), FSB_ERR_RANGE);
    WANT("hidden", create(1000, 0, 32, weights_, scales_, FSB_F16, 0), FSB_ERR_RANGE);
    WANT("hidden", create(1000, FSB_MAX_HIDDEN + 32, 32, weights_, scales_, FSB_F16, 0), FSB_ERR_RANGE);
    WANT("weights", create(1000, 64, 32, nullptr, scales_, FSB_F16, 0), FSB_ERR_INVALID);
    WANT("scales", create(1000, 64, 32, weights_, nullptr, FSB_F16, 0), FSB_ERR_INVALID);
    WANT("scale type", create(1000, 64, 32, weights_, scales_, FSB_F32, 0), FSB_ERR_INVALID);
    WANT("scale alignment", create(1000, 64, 32, weights_, reinterpret_cast<char*>(scales_) + 1, FSB_F16, 0), FSB_ERR_INVALID);
    WANT("flags", create(1000, 64, 32, weights_, scales_, FSB_F16, 2), FSB_ERR_INVALID);
    WANT("out", fsb_head_create(s.h, 1000, 64, 32, weights_, scales_, FSB_F16, 0, nullptr), FSB_ERR_INVALID);
    WANT("handle", fsb_head_create(nullptr, 1000, 64, 32, weights_, scales_, FSB_F16, 0, &head), FSB_ERR_INVALID);
    capturing_ = true;
    rc = create(1000, 64, 32, weights_, scales_, FSB_F16, 0);
    capturing_ = false;
    WANT("captured", rc, FSB_ERR_INVALID);
    WANT("create", create(1000, 64, 32, weights_, scales_, FSB_BF16, FSB_WEIGHTS_ON_HOST), FSB_OK);
    auto logits = [&](const void* x, int type, int n, int64_t ldx, float* to, int64_t ld) { return fsb_head_logits(s.h, head, n, x, type, ldx, to, ld); };
    WANT("fine", logits(hidden_, FSB_F16, 2, 64, out_, 1000), FSB_OK);
    WANT("rows", logits(hidden_, FSB_F16, 0, 64, out_, 1000), FSB_ERR_INVALID);
    WANT("rows", logits(hidden_, FSB_F16, 65536, 64, out_, 1000), FSB_ERR_CAPACITY);
    WANT("type", logits(hidden_, FSB_F32, 2, 64, out_, 1000), FSB_ERR_INVALID);
    WANT("stride", logits(hidden_, FSB_F16, 2, 63, out_, 1000), FSB_ERR_INVALID);
    WANT("stride", logits(hidden_, FSB_F16, 2, 64, out_, 999), FSB_ERR_INVALID);
    WANT("hidden", logits(nullptr, FSB_F16, 2, 64, out_, 1000), FSB_ERR_INVALID);
    WANT("logits", logits(hidden_, FSB_F16, 2, 64, nullptr, 1000), FSB_ERR_INVALID);
    WANT("alignment", logits(reinterpret_cast<char*>(hidden_) + 1, FSB_F16, 2, 64, out_, 1000), FSB_ERR_INVALID);
    WANT("overlap", logits(out_ + 500, FSB_F16, 2, 64, out_, 1000), FSB_ERR_INVALID);
    fsb_head* big = nullptr;
    WANT("create", fsb_head_create(s.h, 1001, 64, 32, std::vector<uint8_t>(1001 * 32).data(), std::vector<uint16_t>(1001 * 2).data(), FSB_F16, 0, &big), FSB_OK);
    WANT("vocabulary of the engine", fsb_sample_hidden(s.h, big, 2, sid, hidden_, FSB_BF16, 64, nullptr, 0, 0, nullptr, tok, 0), FSB_ERR_CAPACITY);
    WANT("rows of the engine", fsb_sample_hidden(s.h, head, 4, sid, hidden_, FSB_BF16, 64, nullptr, 0, 0, nullptr, tok, 0), FSB_ERR_CAPACITY);
    WANT("head", fsb_sample_hidden(s.h, nullptr, 2, sid, hidden_, FSB_BF16, 64, nullptr, 0, 0, nullptr, tok, 0), FSB_ERR_INVALID);
    fsb_destroy(s.h);    // (frees both heads)
    return 0;
}

// A head that is let go while its engine's stream is being captured (by a garbage collector, say): the capture goes on, the head stays.
int captured_free() {
    Setup s(1);
    fsb_head* head = nullptr;
    WANT("create", fsb_head_create(s.h, 1000, 64, 32, weights_, scales_, FSB_F16, 0, &head), FSB_OK);
    capturing_ = true;
    const int rc = fsb_head_free(s.h, head), used = fsb_head_logits(s.h, head, 1, hidden_, FSB_BF16, 64, out_, 1000);
    capturing_ = false;
    WANT("captured", rc, FSB_ERR_INVALID);
    WANT("still there", used, FSB_OK);
    WANT("free", fsb_head_free(s.h, head), FSB_OK);
    return 0;
}

// Launch mode 1 reads logits that are complete before the kernel in front of it starts: our own kernels then start one behind the other.
int modes() {
    Setup s(2);
    fsb_head* head = nullptr;
    WANT("create", fsb_head_create(s.h, 1000, 64, 32, weights_, scales_, FSB_F16, 0, &head), FSB_OK);
    for (int mode = 0; mode < 3; ++mode) {
        fsb_set_launch_overlap(s.h, mode);
        WANT("head", fsb_head_logits(s.h, head, 2, hidden_, FSB_BF16, 64, out_, 1000), FSB_OK);
        WANT("adjust", adjust(s, 2), FSB_OK);
        if (heads_.back().chained != (mode != 1) || heads_.back().scratch_rows != 2) return bad("head", mode, heads_.back().chained, mode != 1);
        if (adjusted_.back()->a.chained != (mode != 1)) return bad("adjust", mode, adjusted_.back()->a.chained, mode != 1);
    }
    return 0;
}

// Settings of the engine that an adjustment cannot compute with, and what does not need one is sampled all the same.
int ranges() {
    Setup s(2);
    int32_t tok[2];
    fsb_head* head = nullptr;
    WANT("create", fsb_head_create(s.h, 1000, 64, 32, weights_, scales_, FSB_F16, 0, &head), FSB_OK);
    auto sampled = [&] { return fsb_sample_batch_adjusted(s.h, 2, s.sid.data(), rows_, FSB_F32, 1000, 1000, nullptr, 0, 0, nullptr, tok, 0); };
    auto hidden = [&](const uint32_t* masks) { return fsb_sample_hidden(s.h, head, 2, s.sid.data(), hidden_, FSB_BF16, 64, masks, 1 << 27, 2, nullptr, tok, 0); };
    for (float cap : {1e38f, 1e13f, 1e-13f, 1e-45f}) {
        fsb_set_softcap(s.h, cap);
        WANT("adjust", adjust(s, 2), FSB_ERR_RANGE);
        WANT("sample", sampled(), FSB_ERR_RANGE);
        WANT("masked", hidden(masks_), FSB_ERR_RANGE);
        WANT("plain", hidden(nullptr), FSB_OK);
    }
    for (float cap : {1e12f, 30.0f, 1e-12f, 0.0f}) {
        fsb_set_softcap(s.h, cap);
        WANT("adjust", adjust(s, 2), FSB_OK);
    }
    for (int32_t past : {0, 1, 1000}) {
        fsb_set_vocab_offset(s.h, INT32_MAX - 1000 + past);
        WANT("offset", adjust(s, 2), past ? FSB_ERR_RANGE : FSB_OK);
        if (past) WANT("offset", hidden(masks_), FSB_ERR_RANGE);
    }
    return 0;
}
}  // namespace

int main(int argc, char** argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    const int rc = what == "settings" ? settings() : what == "regions" ? regions() : what == "sampling" ? sampling() : what == "head" ? head()
                   : what == "refusals" ? refusals() : what == "ranges" ? ranges() : what == "captured_free" ? captured_free() : what == "modes" ? modes() : 2;
    if (rc == 0) std::puts("ok");
    return rc;
}
