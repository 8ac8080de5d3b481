"""What the serving operators refuse is decided on the host, before anything is enqueued: a small driver calls them beneath the context,
without a device, and every call that the documentation rules out has to come back with a status and a text."""
import os
import subprocess


from powerserve_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = r"""
#include "powerserve_b200/csrc/ps_serve.h"
#include <cstdio>
#include <cstring>
#include <functional>

static int no_memory(void *, size_t, void **) { return PS_CUDA_ERR_OOM; }
static int bad = 0;
alignas(16) static float mem[4096];

static void expect(const char *name, int want, const char *text, std::function<int(PsServeCall *)> f) {
    PsServeCall c{};
    c.workspace = no_memory;
    c.n_sm = 148;
    const int rc = f(&c);
    const bool ok = rc == want && (!text || strstr(c.msg, text)) && c.launches == 0;
    if (!ok) { bad++; printf("%s: status %d, text '%s', launches %lld\n", name, rc, c.msg, (long long)c.launches); }
}

int main() {
    const int I = PS_CUDA_ERR_INVALID, U = PS_CUDA_ERR_UNSUPPORTED;
    ps_cuda_cache good{};
    good.k = good.v = mem; good.weight = good.weight_to = mem; good.pos = good.pos_to = reinterpret_cast<int32_t *>(mem);
    good.n_ctx = 16; good.n_kv = 12; good.n_tok = 2; good.n_keep = 8;
    auto attn = [&](const char *name, int want, const char *text, std::function<void(ps_cuda_cache &)> change, int hs = 32, int H = 4, int G = 2, int type = 0, float *out = mem) {
        ps_cuda_cache s = good;
        change(s);
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_attn_tree(c, out, mem, &s, 1, type, hs, H, G, nullptr, 1.f); });
    };
    auto evict = [&](const char *name, int want, const char *text, std::function<void(ps_cuda_cache &)> change, int sink = 0, int recent = 0, int hs = 32, int G = 2, int type = 0) {
        ps_cuda_cache s = good;
        change(s);
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_kv_evict(c, &s, 1, type, hs, G, sink, recent); });
    };
    auto none = [](ps_cuda_cache &) {};
    attn("a call that is right asks for memory", PS_CUDA_ERR_OOM, nullptr, none);
    attn("no tokens: nothing to do", 0, nullptr, [](ps_cuda_cache &s) { s.n_tok = 0; });
    attn("more filled than there are", I, "holds", [](ps_cuda_cache &s) { s.n_kv = 17; });
    attn("filled below zero", I, "holds", [](ps_cuda_cache &s) { s.n_kv = -1; s.n_tok = 0; });
    attn("no slots at all", I, "holds", [](ps_cuda_cache &s) { s.n_ctx = 0; });
    attn("more slots than are taken", U, "slots", [](ps_cuda_cache &s) { s.n_ctx = (1 << 30) + 1; });
    attn("tokens below zero", I, "brings", [](ps_cuda_cache &s) { s.n_tok = -1; });
    attn("more tokens than filled", I, "brings", [](ps_cuda_cache &s) { s.n_tok = 13; });
    attn("too many tokens", U, "brings", [](ps_cuda_cache &s) { s.n_ctx = s.n_kv = 1000; s.n_tok = PS_CUDA_TREE_TOKENS + 1; });
    attn("no keys", I, "no rows", [](ps_cuda_cache &s) { s.k = nullptr; });
    attn("odd address", I, "aligned", [](ps_cuda_cache &s) { s.v = reinterpret_cast<char *>(mem) + 1; });
    attn("odd weights", I, "aligned", [](ps_cuda_cache &s) { s.weight = reinterpret_cast<float *>(reinterpret_cast<char *>(mem) + 2); });
    attn("head size", U, "head size", none, 33);
    attn("head size above", U, "head size", none, 288);
    attn("head size zero", U, "head size", none, 0);
    attn("heads", U, "heads", none, 32, 5);
    attn("heads that share", U, "heads", none, 32, 66);
    attn("no heads", U, "heads", none, 32, 0);
    attn("kv heads", I, "kv heads", none, 32, 4, 0);
    attn("type", U, "cache type", none, 32, 4, 2, 8);
    attn("no output", I, "null", none, 32, 4, 2, 0, nullptr);
    expect("no caches", I, "no caches", [&](PsServeCall *c) { return ps_serve_attn_tree(c, mem, mem, nullptr, 1, 0, 32, 4, 2, nullptr, 1.f); });
    expect("caches below zero", I, "no caches", [&](PsServeCall *c) { return ps_serve_attn_tree(c, mem, mem, &good, -1, 0, 32, 4, 2, nullptr, 1.f); });
    ps_cuda_cache two[2] = {good, good};
    expect("weights gathered twice", I, "same array", [&](PsServeCall *c) { return ps_serve_attn_tree(c, mem, mem, two, 2, 0, 32, 4, 2, nullptr, 1.f); });
    expect("a cache cut twice", I, "share an array", [&](PsServeCall *c) { return ps_serve_kv_evict(c, two, 2, 0, 32, 2, 0, 0); });
    { // caches of their own, one of whose arrays another one reads or writes
        ps_cuda_cache own[2] = {good, good};
        own[0].n_ctx = own[0].n_kv = own[1].n_ctx = own[1].n_kv = 100;
        for (int i = 0; i < 2; i++) {
            char *at = reinterpret_cast<char *>(mem) + 64 * i;
            own[i].k = at; own[i].v = at + 8; own[i].weight = reinterpret_cast<float *>(at + 16); own[i].weight_to = reinterpret_cast<float *>(at + 24);
            own[i].pos = reinterpret_cast<int32_t *>(at + 32); own[i].pos_to = reinterpret_cast<int32_t *>(at + 40);
        }
        auto both = [&](PsServeCall *c) { return ps_serve_kv_evict(c, own, 2, 0, 32, 2, 1, 1); };
        expect("caches of their own ask for memory", PS_CUDA_ERR_OOM, nullptr, both);
        own[1].weight = own[0].weight; own[1].pos = own[0].pos;
        expect("what is only read is shared", PS_CUDA_ERR_OOM, nullptr, both);
        own[1].pos = own[0].pos_to;
        expect("positions that another cache writes", I, "share an array", both);
        own[1].pos = own[0].pos; own[1].pos_to = own[0].pos_to;
        expect("positions written twice", I, "share an array", both);
        own[1].pos_to = reinterpret_cast<int32_t *>(reinterpret_cast<char *>(mem) + 104); own[1].v = own[0].v;
        expect("one V for two", I, "share an array", both);
    }
    expect("nobody", 0, nullptr, [&](PsServeCall *c) { return ps_serve_attn_tree(c, mem, mem, nullptr, 0, 0, 32, 4, 2, nullptr, 1.f); });

    evict("a call that is right asks for memory", PS_CUDA_ERR_OOM, nullptr, [](ps_cuda_cache &s) { s.n_ctx = s.n_kv = 100; }, 1, 1);
    evict("keeps more than there are", I, "keeps", [](ps_cuda_cache &s) { s.n_keep = 13; });
    evict("keeps below zero", I, "keeps", [](ps_cuda_cache &s) { s.n_keep = -1; });
    evict("no weights", I, "gathered", [](ps_cuda_cache &s) { s.weight = nullptr; });
    evict("no new weights", I, "gathered", [](ps_cuda_cache &s) { s.weight_to = nullptr; });
    evict("positions without new ones", I, "together", [](ps_cuda_cache &s) { s.pos_to = nullptr; });
    evict("new positions alone", I, "together", [](ps_cuda_cache &s) { s.pos = nullptr; });
    evict("latest without positions", I, "positions", [](ps_cuda_cache &s) { s.pos = s.pos_to = nullptr; }, 0, 1);
    evict("first without positions", I, "positions", [](ps_cuda_cache &s) { s.pos = s.pos_to = nullptr; }, 1, 0);
    evict("hidden slots", U, "hidden", [](ps_cuda_cache &s) { s.hidden = reinterpret_cast<uint8_t *>(mem); });
    evict("first below zero", I, "first", none, -1, 0);
    evict("latest below zero", I, "latest", none, 0, -1);
    evict("head size", U, "head size", none, 0, 0, 40);
    evict("type", U, "cache type", none, 0, 0, 32, 2, 1);
    expect("nobody", 0, nullptr, [&](PsServeCall *c) { return ps_serve_kv_evict(c, nullptr, 0, 0, 32, 2, 0, 0); });

    int32_t *ids = reinterpret_cast<int32_t *>(mem);
    const ps_cuda_sampler *set = reinterpret_cast<ps_cuda_sampler *>(mem);
    auto samp = [&](const char *name, const char *text, int64_t stride, int64_t vocab, int64_t rows, int32_t *i = nullptr, const float *lg = mem, const ps_cuda_sampler *s = nullptr, const float *u = mem) {
        expect(name, I, text, [&](PsServeCall *c) { return ps_serve_sample(c, i, mem, lg, stride, vocab, rows, s, u); });
    };
    samp("no vocabulary", "rows of", 8, 0, 1, ids, mem, set);
    samp("vocabulary below zero", "rows of", 8, -3, 1, ids, mem, set);
    samp("vocabulary above", "rows of", 1 << 19, (1 << 18) + 1, 1, ids, mem, set);
    samp("rows that overlap", "rows of", 7, 8, 1, ids, mem, set);
    samp("rows below zero", "rows of", 8, 8, -1, ids, mem, set);
    samp("no ids", "null", 8, 8, 1, nullptr, mem, set);
    samp("no logits", "null", 8, 8, 1, ids, nullptr, set);
    samp("no settings", "null", 8, 8, 1, ids, mem, nullptr);
    samp("no numbers", "null", 8, 8, 1, ids, mem, set, nullptr);
    samp("odd logits", "aligned", 8, 8, 1, ids, reinterpret_cast<float *>(reinterpret_cast<char *>(mem) + 1), set);
    expect("no rows", 0, nullptr, [&](PsServeCall *c) { return ps_serve_sample(c, ids, mem, mem, 8, 8, 0, set, mem); });
    printf(bad ? "%d wrong\n" : "all refused\n", bad);
    return bad != 0;
}
"""


def test_every_call_that_is_ruled_out_is_refused(tmp_path):
    lib = build.build()
    src, exe = tmp_path / "driver.cpp", tmp_path / "driver"
    src.write_text(DRIVER)
    cuda = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))
    cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-I" + ROOT, "-I" + os.path.join(cuda, "include"), str(src), lib, "-Wl,-rpath," + os.path.dirname(lib),
           "-L" + os.path.join(cuda, "lib64"), "-Wl,-rpath," + os.path.join(cuda, "lib64"), "-lcudart", "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
