// Host-side exercise of the C ABI's argument checks and launch planning, built
// with AddressSanitizer and UndefinedBehaviorSanitizer on the host code of
// libnqamd (build_and_run.sh). It runs only where no GPU is visible: every call
// either returns an argument error before any device work, or plans its launch
// (descriptor checks, geometry, tile and wave choice, kernel-argument packing)
// and gets NQ_ERR_LAUNCH from the runtime. The fake device buffers below are
// host allocations that nothing dereferences on the host.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "nqamd.h"
#include "nqamd_shell.h"

namespace {

int failures = 0;

void expect(bool ok, const char* what, int got) {
    if (!ok) {
        std::fprintf(stderr, "FAIL %s (status %d)\n", what, got);
        ++failures;
    }
}

// A status from a call that reaches the launch without a device.
bool launch_refused(int st) { return st == NQ_ERR_LAUNCH || st == NQ_ERR_DEVICE; }

struct Buffer {
    void* p = nullptr;
    explicit Buffer(size_t bytes) { p = std::aligned_alloc(256, (bytes + 255) / 256 * 256); }
    ~Buffer() { std::free(p); }
};

nq_linear_desc desc_for(int64_t in, int64_t out, int64_t rank, const Buffer& words, const Buffer& scales,
                        const Buffer& tiles, int64_t tiles_bytes) {
    nq_linear_desc d;
    std::memset(&d, 0, sizeof(d));
    d.in_features = in;
    d.out_features = out;
    d.rank = rank;
    d.right_words = static_cast<const int32_t*>(words.p);
    d.left_words = static_cast<const int32_t*>(words.p);
    d.scale_pre = scales.p;
    d.scale_mid = scales.p;
    d.scale_post = scales.p;
    d.scale_dtype = NQ_DTYPE_F16;
    d.bias_dtype = NQ_DTYPE_F16;
    d.tiles = tiles.p;
    d.tiles_bytes = tiles_bytes;
    d.decode_launch = NQ_DECODE_SPLIT;
    d.prefill_operands = NQ_PREFILL_FP16;
    return d;
}

// A call's workspace, or an alignment's worth where it needs none.
Buffer workspace(int64_t bytes) { return Buffer(static_cast<size_t>(bytes > 0 ? bytes : 256)); }

// Ragged batches over the 8-bit paged cache: sizes at their limits and odd ones
// through every plan, argument errors, and calls up to their launches.
void serving_calls() {
    constexpr int64_t kMost32 = 0x7fffffff, kMost64 = INT64_MAX;
    const int64_t counts[] = {-1, 0, 1, 2, 3, 17, 64, 65, 1000, 65535, 65536, 1 << 20, (1 << 24) - 32, 1 << 24, 0x3fffffff,
                              kMost32 - 1, kMost32, kMost64};
    for (const int64_t tokens : counts)
        for (const int64_t size : counts) {
            for (const int32_t group : {0, 32, 64, 128})
                for (const int64_t ins : {int64_t{0}, int64_t{32}, int64_t{1152}, int64_t{10240}, int64_t{1} << 24, kMost64})
                    expect(nq_int4_projection_workspace_bytes(tokens, size, ins, group) >= -1, "4-bit workspace", 0);
            expect(nq_int4_projection_partials(size) >= -1, "4-bit partials", 0);
            for (const int64_t batch : counts)
                for (const int32_t page : {0, 16, 128}) {
                    for (const int32_t heads : {0, 4, 65535})
                        expect(nq_paged_evict_workspace_bytes(batch, heads, page, size, tokens) >= -1, "evict workspace", 0);
                    for (const int32_t kv_heads : {1, 8})
                        for (const int32_t head_dim : {64, 96, 128, 256}) {
                            const int64_t paged = nq_paged_attention_workspace_bytes(tokens, batch, 32, kv_heads, head_dim, page, size);
                            expect(paged >= -1 && paged <= int64_t{1} << 30, "paged attention workspace", 0);
                            for (const int64_t shared : {int64_t{-1}, int64_t{0}, int64_t{1000}, kMost64}) {
                                const int64_t w = nq_shared_attention_workspace_bytes(tokens, batch, 32, kv_heads, head_dim, page, size, shared);
                                expect(w >= -1 && w <= int64_t{1} << 30, "shared attention workspace", 0);
                            }
                        }
                }
            for (const int32_t top : {-1, 0, 5, 32, 33})
                expect(nq_token_logprobs_workspace_bytes(tokens, size, top) >= -1, "logprobs workspace", 0);
        }

    Buffer cache(1 << 20), scales(1 << 16), lens(1 << 16), table(1 << 16), x(1 << 20), y(1 << 20), into(1 << 16), rows(1 << 20);
    const auto fp = [](const Buffer& b) { return static_cast<float*>(b.p); };
    const auto ints = [](const Buffer& b) { return static_cast<int32_t*>(b.p); };
    const int dtypes[] = {NQ_DTYPE_F32, NQ_DTYPE_F16, NQ_DTYPE_BF16};
    for (const int32_t head_dim : {64, 128, 256})
        for (const int32_t page : {16, 32, 64, 128})
            for (const int64_t batch : {1, 3, 65, 300})
                for (const int64_t tokens : {1, 40, 700, 5000})
                    for (const int64_t pages : {3, 200, 9000}) {
                        nq_paged_kv kv;
                        std::memset(&kv, 0, sizeof(kv));
                        kv.k_pages = kv.v_pages = cache.p;
                        kv.k_scales = kv.v_scales = fp(scales);
                        kv.num_pages = 1000000;
                        kv.kv_heads = 4;
                        kv.head_dim = head_dim;
                        kv.page_size = page;
                        kv.page_table = ints(table);
                        kv.table_pages = pages;
                        kv.query_starts = kv.context_lens = ints(lens);
                        kv.batch = batch;
                        const int type = dtypes[(batch + tokens) % 3];
                        int st = nq_paged_append(x.p, x.p, x.p, type, tokens, 16, scales.p, scales.p, NQ_DTYPE_F32, 1e-6f, fp(y), fp(y),
                                                 40000, &kv, y.p, type, nullptr);
                        expect(launch_refused(st), "paged append", st);
                        st = nq_paged_append_at(x.p, x.p, x.p, type, tokens, 16, nullptr, nullptr, NQ_DTYPE_F32, 1e-6f, fp(y), fp(y),
                                                kMost64, &kv, ints(lens), y.p, type, nullptr);
                        expect(launch_refused(st), "paged append at", st);
                        int64_t need = nq_paged_attention_workspace_bytes(tokens, batch, 16, 4, head_dim, page, pages);
                        {
                            const Buffer ws = workspace(need);
                            st = nq_paged_attention(x.p, type, tokens, 16, &kv, 0.1f, y.p, type, ws.p, need, nullptr);
                            expect(launch_refused(st), "paged attention", st);
                        }
                        for (const int64_t shared : {int64_t{0}, page * pages / 2, page * pages}) {
                            need = nq_shared_attention_workspace_bytes(tokens, batch, 16, 4, head_dim, page, pages, shared);
                            const Buffer ws = workspace(need);
                            st = nq_shared_attention(x.p, type, tokens, 16, &kv, shared, 0.1f, y.p, type, fp(y), ws.p, need, nullptr);
                            expect(launch_refused(st), "shared attention", st);
                            if (need > 0) {
                                st = nq_shared_attention(x.p, type, tokens, 16, &kv, shared, 0.1f, y.p, type, nullptr, ws.p, need - 1, nullptr);
                                expect(st == NQ_ERR_WORKSPACE, "shared attention short workspace", st);
                            }
                        }
                        for (const int64_t first : {int64_t{0}, int64_t{33}, page * pages - 1})
                            expect(launch_refused(nq_attention_weights(x.p, type, tokens, 16, &kv, 0.1f, fp(y), first, fp(y), fp(y), nullptr)),
                                   "attention weights", 0);
                        expect(nq_attention_weights(x.p, type, tokens, 16, &kv, 0.1f, fp(y), page * pages, fp(y), fp(y), nullptr) == NQ_OK,
                               "attention weights of no row", 0);
                        for (const int64_t budget : {int64_t{1}, int64_t{50}, page * pages, page * pages + 1}) {
                            need = nq_paged_evict_workspace_bytes(batch, 4, page, pages, budget);
                            const Buffer ws = workspace(need);
                            if (need < 0) {  // more pages to move than a launch has workgroups
                                st = nq_paged_evict(&kv, fp(y), ints(into), budget, 0, 0, ints(rows), ints(x), ints(rows), ws.p, 256, nullptr);
                                expect(st == NQ_ERR_SHAPE && batch > 64 && budget > 100000, "evict of a size that it refuses", st);
                                continue;
                            }
                            st = nq_paged_evict(&kv, fp(y), ints(into), budget, budget / 3, budget / 4, ints(rows), ints(x), ints(rows), ws.p, need,
                                                nullptr);
                            expect(launch_refused(st), "evict", st);
                            st = nq_paged_evict(&kv, fp(y), ints(into), budget, budget, 1, ints(rows), ints(x), ints(rows), ws.p, need, nullptr);
                            expect(st == NQ_ERR_SHAPE, "evict more than its budget", st);
                        }
                    }
    expect(nq_paged_append(nullptr, nullptr, nullptr, 0, 1, 1, nullptr, nullptr, 0, 0.0f, nullptr, nullptr, 1, nullptr, nullptr, 0, nullptr) ==
               NQ_ERR_ARGUMENT, "paged append null", 0);
    expect(nq_shared_attention(x.p, 0, 1, 1, nullptr, 0, 0.1f, y.p, 0, nullptr, nullptr, 0, nullptr) == NQ_ERR_ARGUMENT, "shared attention null", 0);
    expect(nq_attention_weights(x.p, 0, 1, 1, nullptr, 0.1f, fp(y), 0, fp(y), fp(y), nullptr) == NQ_ERR_ARGUMENT, "attention weights null", 0);
    expect(nq_paged_evict(nullptr, nullptr, nullptr, 1, 0, 0, nullptr, nullptr, nullptr, nullptr, 0, nullptr) == NQ_ERR_ARGUMENT, "evict null", 0);

    for (const int32_t group : {32, 64, 128})
        for (const int64_t tokens : {1, 2, 5, 11, 31, 256, 65535})
            for (const int64_t outs : {1, 100, 12304, 49268})
                for (const int64_t ins : {32, 1152, 10240, 30912})
                    for (const int x_dtype : dtypes) {
                        const int64_t need = nq_int4_projection_workspace_bytes(tokens, outs, ins, group);
                        expect(need >= 0, "4-bit workspace", 0);
                        const Buffer ws(256);  // not touched on the host
                        int st = nq_int4_projection(x.p, x_dtype, tokens, cache.p, scales.p, dtypes[tokens % 3],
                                                    static_cast<uint8_t*>(scales.p), outs, ins, group, y.p, NQ_DTYPE_BF16,
                                                    tokens == 1 ? rows.p : nullptr, ws.p, need, nullptr);
                        expect(launch_refused(st), "4-bit projection", st);
                        if (need == 0) continue;
                        st = nq_int4_projection(x.p, x_dtype, tokens, cache.p, scales.p, NQ_DTYPE_F16, nullptr, outs, ins, group, y.p, NQ_DTYPE_F32,
                                                nullptr, ws.p, need - 1, nullptr);
                        expect(st == NQ_ERR_WORKSPACE, "4-bit short workspace", st);
                    }
    expect(nq_int4_projection(nullptr, 0, 1, nullptr, nullptr, 0, nullptr, 1, 32, 32, nullptr, 0, nullptr, nullptr, 0, nullptr) == NQ_ERR_ARGUMENT,
           "4-bit null", 0);
    int st = nq_greedy_select_partials(rows.p, 9496, static_cast<int64_t*>(y.p), nullptr, 0, nullptr, nullptr, nullptr);
    expect(launch_refused(st), "greedy select partials", st);
    for (const int64_t count : {int64_t{1}, int64_t{1531}})
        for (const int32_t top : {0, 5, 32}) {
            const int64_t need = nq_token_logprobs_workspace_bytes(count, 151936, top);
            const Buffer ws = workspace(need);
            st = nq_token_logprobs(x.p, NQ_DTYPE_F32, count, 151936, 151936, static_cast<int64_t*>(y.p), top, fp(y), fp(y),
                                   static_cast<int64_t*>(y.p), fp(y), ws.p, need, nullptr);
            expect(launch_refused(st), "token logprobs", st);
        }
}

}  // namespace

int main() {
    nq_device_caps caps;
    if (nq_query_device(0, &caps) == NQ_OK) {
        std::printf("a GPU is visible: this host-only driver runs nothing\n");
        return 77;
    }
    expect(nq_abi_version() > 0, "abi version", 0);
    expect(nq_tiles_header_bytes() > 0, "tiles header", 0);
    for (int s = -20; s <= 1; ++s) expect(nq_status_string(s) != nullptr, "status string", s);

    // Argument errors.
    expect(nq_unpack_signs(nullptr, 1, 1, 1, NQ_DTYPE_F32, nullptr, nullptr) == NQ_ERR_ARGUMENT, "unpack null", 0);
    expect(nq_tiles_bytes(0, 1, 1) < 0 && nq_tiles_bytes(1, 1, -1) < 0, "tiles bytes shape", 0);
    nq_linear_desc bad;
    std::memset(&bad, 0, sizeof(bad));
    expect(nq_linear_workspace_bytes(&bad, 1) == -1, "workspace of empty desc", 0);
    expect(nq_linear(&bad, nullptr, 0, 1, nullptr, 0, nullptr, 0, nullptr) != NQ_OK, "linear empty desc", 0);
    expect(nq_linear_batch(nullptr, 0, nullptr, 0, 1, nullptr, 0, nullptr, nullptr, nullptr) != NQ_OK, "batch null", 0);
    expect(nq_embedding(nullptr, 1, nullptr, NQ_DTYPE_BF16, 1, 8, nullptr, nullptr, nullptr) == NQ_ERR_ARGUMENT,
           "embedding null", 0);
    expect(nq_embedding_slots(nullptr, 1, nullptr, NQ_DTYPE_BF16, 1, 16, nullptr, nullptr, nullptr, nullptr) ==
               NQ_ERR_ARGUMENT, "embedding slots null", 0);
    expect(nq_add_rmsnorm(nullptr, nullptr, 0, nullptr, 0, 1e-6f, 1, 8, nullptr, 0, nullptr) == NQ_ERR_ARGUMENT,
           "add_rmsnorm null", 0);
    expect(nq_silu_mul(nullptr, nullptr, 8, nullptr, NQ_DTYPE_F32, nullptr) != NQ_OK, "silu null", 0);
    expect(nq_greedy_select(nullptr, 1, 8, nullptr, nullptr, 0, nullptr, nullptr, nullptr) == NQ_ERR_ARGUMENT,
           "greedy null", 0);
    expect(nq_decode_attention_workspace_bytes(32, 7, 128, NQ_DTYPE_BF16, 640) == -1, "attention heads", 0);
    expect(nq_output_projection_workspace_bytes(151936, 4096) > 0, "lm_head workspace", 0);
    expect(nq_attention_workspace_bytes(1, 32, 128, 640) > 0, "attention workspace", 0);

    // Launch planning of decode and prefill calls over the Qwen3-8B projection
    // shapes, every token count of the decode range and a few prefill ones.
    const int64_t shapes[][3] = {{4096, 4096, 2048}, {4096, 1024, 819}, {4096, 12288, 3072},
                                 {12288, 4096, 3072}, {1152, 6912, 768}, {35, 17, 5}};
    const int64_t token_counts[] = {1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 40, 64, 300};
    Buffer words(64 << 20), scales(1 << 20), x(64 << 20), y(64 << 20);
    for (const auto& sh : shapes) {
        const int64_t tb = nq_tiles_bytes(sh[0], sh[1], sh[2]);
        expect(tb > 0, "tiles bytes", 0);
        Buffer tiles(static_cast<size_t>(tb));
        for (int launch : {NQ_DECODE_SPLIT, NQ_DECODE_FUSED}) {
            nq_linear_desc d = desc_for(sh[0], sh[1], sh[2], words, scales, tiles, tb);
            d.decode_launch = launch;
            for (int64_t t : token_counts) {
                const int64_t wb = nq_linear_workspace_bytes(&d, t);
                expect(wb >= 0, "workspace bytes", static_cast<int>(wb));
                Buffer ws(static_cast<size_t>(wb > 0 ? wb : 1));
                for (int xd : {NQ_DTYPE_BF16, NQ_DTYPE_F32}) {
                    const int st = nq_linear(&d, x.p, xd, t, y.p, NQ_DTYPE_F32, ws.p, wb, nullptr);
                    expect(launch_refused(st), "linear launch", st);
                }
                const int st2 = nq_linear(&d, x.p, NQ_DTYPE_BF16, t, y.p, NQ_DTYPE_F32, ws.p, wb - 1, nullptr);
                expect(st2 == NQ_ERR_WORKSPACE, "linear short workspace", st2);
            }
        }
    }

    // A batch of the seven Qwen3-8B linears (one call per layer), and the
    // fused one-token forms the decoder uses.
    {
        const int64_t layer[7][3] = {{4096, 4096, 2048}, {4096, 1024, 819}, {4096, 1024, 819}, {4096, 4096, 2048},
                                     {4096, 12288, 3072}, {4096, 12288, 3072}, {12288, 4096, 3072}};
        std::vector<Buffer*> tiles, wss;
        std::vector<nq_linear_desc> descs(7);
        std::vector<const nq_linear_desc*> dp(7);
        std::vector<const void*> xs(7, x.p);
        std::vector<void*> ys(7, y.p), wp(7);
        std::vector<int64_t> wb(7);
        for (int i = 0; i < 7; ++i) {
            const int64_t tb = nq_tiles_bytes(layer[i][0], layer[i][1], layer[i][2]);
            tiles.push_back(new Buffer(static_cast<size_t>(tb)));
            descs[i] = desc_for(layer[i][0], layer[i][1], layer[i][2], words, scales, *tiles.back(), tb);
            dp[i] = &descs[i];
            wb[i] = nq_linear_workspace_bytes(&descs[i], 300);  // the largest token count below
            wss.push_back(new Buffer(static_cast<size_t>(wb[i])));
            wp[i] = wss.back()->p;
        }
        for (int64_t t : token_counts) {
            const int st = nq_linear_batch(dp.data(), 7, xs.data(), NQ_DTYPE_BF16, t, ys.data(), NQ_DTYPE_F32,
                                           wp.data(), wb.data(), nullptr);
            expect(launch_refused(st), "layer batch", st);
        }
        Buffer slots(1 << 16), colscale(1 << 20), residual(1 << 20);
        std::vector<const float*> cs(7, static_cast<const float*>(colscale.p));
        std::vector<const void*> ups(7, residual.p);
        std::vector<float*> res(7, static_cast<float*>(residual.p)), outs(7, static_cast<float*>(slots.p));
        nq_decode_fusion f;
        std::memset(&f, 0, sizeof(f));
        f.input_kind = NQ_INPUT_RMSNORM;
        f.eps = 1e-6f;
        f.col_scales = cs.data();
        f.norm_slots = static_cast<const float*>(slots.p);
        f.norm_slot_count = 256;
        int st = nq_linear_batch_fused(dp.data(), 3, xs.data(), NQ_DTYPE_F32, ys.data(), NQ_DTYPE_F32, wp.data(),
                                       wb.data(), &f, nullptr);
        expect(launch_refused(st), "fused qkv", st);
        f.output_kind = NQ_OUTPUT_SILU_PRODUCT;
        st = nq_linear_batch_fused(dp.data() + 4, 2, xs.data(), NQ_DTYPE_F32, ys.data(), NQ_DTYPE_BF16,
                                   wp.data() + 4, wb.data() + 4, &f, nullptr);
        expect(launch_refused(st), "fused gate/up", st);
        std::memset(&f, 0, sizeof(f));
        f.input_kind = NQ_INPUT_PLAIN;
        f.residuals = res.data();
        f.out_slots = outs.data();
        st = nq_linear_batch_fused(dp.data() + 6, 1, xs.data(), NQ_DTYPE_BF16, ys.data(), NQ_DTYPE_F32,
                                   wp.data() + 6, wb.data() + 6, &f, nullptr);
        expect(launch_refused(st), "fused down", st);
        f.input_kind = NQ_INPUT_SILU_GATE;
        f.ups = ups.data();
        st = nq_linear_batch_fused(dp.data() + 6, 1, xs.data(), NQ_DTYPE_F32, ys.data(), NQ_DTYPE_F32,
                                   wp.data() + 6, wb.data() + 6, &f, nullptr);
        expect(launch_refused(st), "fused gated down", st);
        for (Buffer* b : tiles) delete b;
        for (Buffer* b : wss) delete b;
    }

    // The other entry points, each planned up to its launch with buffers of the
    // sizes it checks (Qwen3-8B geometry where it has one).
    {
        Buffer big(64 << 20), ws(64 << 20), ids(64), pos(64), tok(64), hist(1024), stepb(64), counts(4096);
        int st = nq_embedding(static_cast<const int64_t*>(ids.p), 1, big.p, NQ_DTYPE_BF16, 151936, 4096, nullptr,
                              static_cast<float*>(ws.p), nullptr);
        expect(launch_refused(st), "embedding", st);
        st = nq_embedding_slots(static_cast<const int64_t*>(ids.p), 1, big.p, NQ_DTYPE_BF16, 151936, 4096, nullptr,
                                static_cast<float*>(ws.p), static_cast<float*>(x.p), nullptr);
        expect(launch_refused(st), "embedding slots", st);
        st = nq_embedding_slots(static_cast<const int64_t*>(ids.p), 1, big.p, NQ_DTYPE_BF16, 10, 24, nullptr,
                                static_cast<float*>(ws.p), static_cast<float*>(x.p), nullptr);
        expect(st == NQ_ERR_SHAPE, "embedding slots hidden % 16", st);
        for (int64_t t : {int64_t(1), int64_t(37)}) {
            st = nq_add_rmsnorm(static_cast<float*>(big.p), x.p, NQ_DTYPE_F32, scales.p, NQ_DTYPE_BF16, 1e-6f, t, 4096,
                                y.p, NQ_DTYPE_BF16, nullptr);
            expect(launch_refused(st), "add_rmsnorm", st);
        }
        st = nq_silu_mul(static_cast<const float*>(x.p), static_cast<const float*>(y.p), 12288, ws.p, NQ_DTYPE_BF16,
                         nullptr);
        expect(launch_refused(st), "silu_mul", st);
        const int64_t pw = nq_output_projection_workspace_bytes(151936, 4096);
        st = nq_output_projection(x.p, NQ_DTYPE_F32, big.p, 151936, 4096, static_cast<float*>(y.p), ws.p, pw, nullptr);
        expect(launch_refused(st), "output projection", st);
        st = nq_greedy_select(ws.p, 151936, 4096, static_cast<int64_t*>(tok.p), static_cast<int64_t*>(hist.p), 128,
                              static_cast<int32_t*>(stepb.p), static_cast<int32_t*>(pos.p), nullptr);
        expect(launch_refused(st), "greedy select", st);
        for (int64_t mp : {int64_t(128), int64_t(640), int64_t(1100)}) {
            for (int hd : {64, 128}) {
                const int64_t dw = nq_decode_attention_workspace_bytes(32, 8, hd, NQ_DTYPE_BF16, mp);
                expect(dw > 0, "decode attention workspace", static_cast<int>(dw));
                st = nq_decode_attention(static_cast<const float*>(x.p), static_cast<const float*>(x.p),
                                         static_cast<const float*>(x.p), 32, 8, hd, scales.p, scales.p, NQ_DTYPE_BF16,
                                         1e-6f, static_cast<const float*>(big.p), static_cast<const float*>(big.p),
                                         static_cast<const int32_t*>(pos.p), mp, ws.p, y.p, NQ_DTYPE_BF16, 0.088f,
                                         x.p, NQ_DTYPE_F32, words.p, dw, nullptr);
                expect(launch_refused(st), "decode attention", st);
                st = nq_decode_attention_partials(static_cast<const float*>(x.p), static_cast<const float*>(x.p),
                                                  static_cast<const float*>(x.p), 32, 8, hd, scales.p, scales.p,
                                                  NQ_DTYPE_BF16, 1e-6f, static_cast<const float*>(big.p),
                                                  static_cast<const float*>(big.p), static_cast<const int32_t*>(pos.p),
                                                  mp, ws.p, y.p, NQ_DTYPE_BF16, 0.088f, words.p, dw, nullptr);
                expect(launch_refused(st), "decode attention partials", st);
            }
            for (int64_t t : {int64_t(1), int64_t(17), int64_t(64)}) {
                const int64_t aw = nq_attention_workspace_bytes(t, 32, 128, mp);
                st = nq_qk_norm_rope_cache(static_cast<const float*>(x.p), static_cast<const float*>(x.p),
                                           static_cast<const float*>(x.p), t, 32, 8, 128, scales.p, scales.p,
                                           NQ_DTYPE_BF16, 1e-6f, static_cast<const float*>(big.p),
                                           static_cast<const float*>(big.p), static_cast<const int32_t*>(pos.p), mp,
                                           static_cast<float*>(y.p), ws.p, words.p, NQ_DTYPE_BF16, nullptr);
                expect(launch_refused(st), "qk norm rope cache", st);
                st = nq_attention(static_cast<const float*>(x.p), ws.p, words.p, NQ_DTYPE_BF16, t, 32, 8, 128,
                                  static_cast<const int32_t*>(pos.p), mp, 0.088f, y.p, NQ_DTYPE_BF16, big.p, aw,
                                  nullptr);
                expect(launch_refused(st), "attention", st);
            }
        }
        st = nq_unpack_signs(static_cast<const int32_t*>(words.p), 3072, 819, 26, NQ_DTYPE_BF16, ws.p, nullptr);
        expect(launch_refused(st), "unpack", st);
        st = nq_count_bad_padding(static_cast<const int32_t*>(words.p), 3072, 819, 26,
                                  static_cast<int32_t*>(counts.p), nullptr);
        expect(launch_refused(st), "bad padding", st);
        st = nq_transpose_signs(static_cast<const int32_t*>(words.p), 819, 3072, static_cast<int32_t*>(ws.p),
                                nullptr);
        expect(launch_refused(st) || st == NQ_OK, "transpose signs", st);
        const int64_t tb = nq_tiles_bytes(4096, 1024, 819);
        Buffer tiles(static_cast<size_t>(tb));
        nq_linear_desc d = desc_for(4096, 1024, 819, words, scales, tiles, tb);
        st = nq_prepare_tiles(&d, tiles.p, tb, nullptr);
        expect(launch_refused(st), "prepare tiles", st);
        for (int64_t t : {int64_t(1), int64_t(4), int64_t(16)}) {
            st = nq_linear_static(&d, x.p, NQ_DTYPE_BF16, t, y.p, NQ_DTYPE_F32, nullptr);
            expect(st != NQ_OK, "linear static", st);
        }
        st = nq_decode_mixed_v_words(nullptr, 0, nullptr, 0, nullptr, 819, 4096, nullptr, nullptr, nullptr);
        expect(st != NQ_OK, "mixed-v null", st);
        st = nq_decode_product_codebook_words(nullptr, 0, nullptr, 0, nullptr, nullptr, 819, 4096, nullptr, nullptr);
        expect(st != NQ_OK, "product codebook null", st);
        st = nq_read_stream(big.p, 1 << 20, static_cast<uint32_t*>(counts.p), 64, nullptr);
        expect(launch_refused(st), "read stream", st);
    }

    serving_calls();

    std::printf("%s: %d failed checks\n", failures ? "FAILED" : "ok", failures);
    return failures ? 1 : 0;
}
