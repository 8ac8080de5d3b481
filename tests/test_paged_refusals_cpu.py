"""What the operators on paged caches and the verification of drafted tokens refuse is decided on the host, before anything is enqueued: a small driver calls them beneath the context, without a device; and what
their Python forms refuse before that."""
import os
import subprocess

import numpy as np
import pytest

from powerserve_b200 import build, capi

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
template <typename T> T *odd(int by = 1) { return reinterpret_cast<T *>(reinterpret_cast<char *>(mem) + by); }

int main() {
    const int I = PS_CUDA_ERR_INVALID, U = PS_CUDA_ERR_UNSUPPORTED;
    ps_cuda_pages good{};
    good.codes = reinterpret_cast<int8_t *>(mem); good.scales = mem; good.refs = reinterpret_cast<int32_t *>(mem);
    good.n_layers = 2; good.n_pages = 10; good.page_tokens = 16; good.n_kv_heads = 2; good.head_size = 64;
    ps_cuda_paged_seq one{};
    one.table = reinterpret_cast<int32_t *>(mem); one.n_kv = 20; one.n_tok = 2; one.n_table = 2;

    // what all of them check of a cache
    auto cache = [&](const char *name, int want, const char *text, std::function<void(ps_cuda_pages &)> change) {
        ps_cuda_pages p = good;
        change(p);
        ps_cuda_page_edit e{};
        ps_cuda_page_move m{};
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_rows(c, true, &p, 0, mem, mem, 0, &one, 1); });
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_rows(c, false, &p, 0, mem, mem, 0, &one, 1); });
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_attn(c, &p, 0, mem, mem, 0, &one, 1, 4, nullptr, 1.f); });
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_edit(c, &p, &e, 1, nullptr); });
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_compact(c, &p, &m, 1); });
    };
    for (int t : {0, -16, 8, 17, 48, 256}) cache("page", U, "pages of", [&](ps_cuda_pages &p) { p.page_tokens = t; });
    for (int t : {0, -32, 33, 48, 288}) cache("head size", U, "head size", [&](ps_cuda_pages &p) { p.head_size = t; });
    for (int t : {0, -1, 1025}) cache("kv heads", I, "kv heads", [&](ps_cuda_pages &p) { p.n_kv_heads = t; });
    for (int t : {0, -1, 4097}) cache("layers", I, "layers", [&](ps_cuda_pages &p) { p.n_layers = t; });
    for (int t : {0, -1, (1 << 26) + 1}) cache("pages", I, "pages", [&](ps_cuda_pages &p) { p.n_pages = t; });
    cache("no codes", I, "without codes", [](ps_cuda_pages &p) { p.codes = nullptr; });
    cache("no scales", I, "without codes", [](ps_cuda_pages &p) { p.scales = nullptr; });
    cache("codes at odd places", I, "aligned", [](ps_cuda_pages &p) { p.codes = odd<int8_t>(8); });
    cache("scales at odd places", I, "aligned", [](ps_cuda_pages &p) { p.scales = odd<float>(2); });

    auto seq = [&](const char *name, int want, const char *text, std::function<void(ps_cuda_paged_seq &)> change, int layer = 0, int type = 0, float *k = mem, float *v = mem) {
        ps_cuda_paged_seq s = one;
        change(s);
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_rows(c, true, &good, layer, k, v, type, &s, 1); });
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_attn(c, &good, layer, k, v, type, &s, 1, 4, nullptr, 1.f); });
    };
    auto none = [](ps_cuda_paged_seq &) {};
    seq("no tokens: nothing to do", 0, nullptr, [](ps_cuda_paged_seq &s) { s.n_tok = 0; s.table = nullptr; });
    seq("filled below zero", I, "holds", [](ps_cuda_paged_seq &s) { s.n_kv = -1; });
    seq("more than are taken", I, "holds", [](ps_cuda_paged_seq &s) { s.n_kv = (1 << 30) + 1; });
    seq("more tokens than slots", I, "tokens", [](ps_cuda_paged_seq &s) { s.n_tok = 21; });
    seq("tokens below zero", I, "tokens", [](ps_cuda_paged_seq &s) { s.n_tok = -1; });
    seq("no table", I, "no table", [](ps_cuda_paged_seq &s) { s.table = nullptr; });
    seq("odd table", I, "no table", [](ps_cuda_paged_seq &s) { s.table = odd<int32_t>(); });
    seq("short table", I, "its table", [](ps_cuda_paged_seq &s) { s.n_table = 1; });
    seq("layer", I, "layer", none, 2);
    seq("layer below zero", I, "layer", none, -1);
    seq("type", U, "type", none, 0, 8);
    seq("no rows", I, "null", none, 0, 0, nullptr, nullptr);
    seq("one of two", I, "null", none, 0, 0, nullptr);
    seq("odd rows", I, "aligned", none, 0, 0, odd<float>(2));
    seq("odd rows of bfloat16", I, "aligned", none, 0, 30, mem, odd<float>(1));
    expect("nothing to load", I, "null", [&](PsServeCall *c) { return ps_serve_paged_rows(c, false, &good, 0, nullptr, nullptr, 0, &one, 1); });
    expect("no sequences", I, "no sequences", [&](PsServeCall *c) { return ps_serve_paged_rows(c, true, &good, 0, mem, mem, 0, nullptr, 1); });
    expect("sequences below zero", I, "no sequences", [&](PsServeCall *c) { return ps_serve_paged_attn(c, &good, 0, mem, mem, 0, &one, -1, 4, nullptr, 1.f); });
    expect("no cache", I, "no cache", [&](PsServeCall *c) { return ps_serve_paged_attn(c, nullptr, 0, mem, mem, 0, &one, 1, 4, nullptr, 1.f); });
    for (int H : {0, -2, 3, 66}) expect("heads", U, "heads", [&](PsServeCall *c) { return ps_serve_paged_attn(c, &good, 0, mem, mem, 0, &one, 1, H, nullptr, 1.f); });
    {
        ps_cuda_paged_seq s = one;
        s.n_kv = s.n_tok = PS_CUDA_TREE_TOKENS + 1; s.n_table = 17;
        expect("too many tokens", U, "brings", [&](PsServeCall *c) { return ps_serve_paged_attn(c, &good, 0, mem, mem, 0, &s, 1, 4, nullptr, 1.f); });
        s.n_kv = s.n_tok = INT32_MAX / 1024 + 1; s.n_table = 1 << 20;
        expect("far too many rows", U, "in one call", [&](PsServeCall *c) { return ps_serve_paged_rows(c, true, &good, 0, mem, mem, 0, &s, 1); });
    }
    expect("nobody", 0, nullptr, [&](PsServeCall *c) { return ps_serve_paged_attn(c, &good, 0, nullptr, nullptr, 0, nullptr, 0, 4, nullptr, 1.f); });

    // edits
    ps_cuda_page_edit grow{};
    grow.table = reinterpret_cast<int32_t *>(mem); grow.n_old = 20; grow.n_new = 40; grow.n_table = 3;
    auto edit = [&](const char *name, int want, const char *text, std::function<void(ps_cuda_page_edit &)> change, int32_t *held = nullptr) {
        ps_cuda_page_edit e = grow;
        change(e);
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_edit(c, &good, &e, 1, held); });
    };
    edit("a call that is right asks for memory", PS_CUDA_ERR_OOM, nullptr, [](ps_cuda_page_edit &) {});
    edit("held below zero", I, "tokens", [](ps_cuda_page_edit &e) { e.n_old = -1; });
    edit("wanted below zero", I, "tokens", [](ps_cuda_page_edit &e) { e.n_new = -1; });
    edit("wanted above", I, "tokens", [](ps_cuda_page_edit &e) { e.n_new = (1 << 30) + 1; });
    edit("short table", I, "its table", [](ps_cuda_page_edit &e) { e.n_table = 2; });
    edit("table too short for what it held", I, "its table", [](ps_cuda_page_edit &e) { e.n_new = 1; e.n_table = 1; });
    edit("no table", I, "no table", [](ps_cuda_page_edit &e) { e.table = nullptr; });
    edit("odd table", I, "no table", [](ps_cuda_page_edit &e) { e.table = odd<int32_t>(); });
    edit("odd beginning", I, "no table", [](ps_cuda_page_edit &e) { e.from = odd<int32_t>(2); });
    edit("shares and shrinks", I, "shares", [](ps_cuda_page_edit &e) { e.from = reinterpret_cast<int32_t *>(mem + 64); e.n_new = 10; });
    edit("begins as itself", I, "as itself", [](ps_cuda_page_edit &e) { e.from = e.table; });
    edit("odd answer", I, "aligned", [](ps_cuda_page_edit &) {}, odd<int32_t>());
    {
        ps_cuda_page_edit two[2] = {grow, grow};
        expect("a table twice", I, "one table", [&](PsServeCall *c) { return ps_serve_paged_edit(c, &good, two, 2, nullptr); });
        ps_cuda_page_edit chain[3] = {grow, grow, grow}; // a table begins as one that begins as a third
        for (int i = 0; i < 3; i++) { chain[i].table = reinterpret_cast<int32_t *>(mem) + 64 * (i + 1); chain[i].from = reinterpret_cast<int32_t *>(mem); }
        expect("three begin as one", PS_CUDA_ERR_OOM, nullptr, [&](PsServeCall *c) { return ps_serve_paged_edit(c, &good, chain, 3, nullptr); });
        for (int by : {0, 2}) {
            chain[1].from = chain[by].table;
            expect("a chain", I, "begins anew", [&](PsServeCall *c) { return ps_serve_paged_edit(c, &good, chain, 3, nullptr); });
        }
        ps_cuda_pages p = good;
        p.refs = nullptr;
        expect("no counts", I, "without refs", [&](PsServeCall *c) { return ps_serve_paged_edit(c, &p, two, 1, nullptr); });
        p.refs = odd<int32_t>(2);
        expect("odd counts", I, "aligned", [&](PsServeCall *c) { return ps_serve_paged_edit(c, &p, two, 1, nullptr); });
        expect("no edits", I, "no edits", [&](PsServeCall *c) { return ps_serve_paged_edit(c, &good, nullptr, 1, nullptr); });
        expect("edits below zero", I, "no edits", [&](PsServeCall *c) { return ps_serve_paged_edit(c, &good, two, -1, nullptr); });
        expect("too many edits", U, "edits", [&](PsServeCall *c) { return ps_serve_paged_edit(c, &good, two, PS_CUDA_EDITS + 1, nullptr); });
        expect("none", 0, nullptr, [&](PsServeCall *c) { return ps_serve_paged_edit(c, &good, nullptr, 0, nullptr); });
    }

    // moves
    ps_cuda_page_move some{};
    some.table = some.keep = reinterpret_cast<int32_t *>(mem); some.first = 4; some.n_kv = 30; some.n_keep = 5; some.n_table = 2;
    auto move = [&](const char *name, int want, const char *text, std::function<void(ps_cuda_page_move &)> change) {
        ps_cuda_page_move m = some;
        change(m);
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_paged_compact(c, &good, &m, 1); });
    };
    move("first below zero", I, "slot", [](ps_cuda_page_move &m) { m.first = -1; });
    move("first behind the last", I, "slot", [](ps_cuda_page_move &m) { m.first = 31; });
    move("filled above", I, "slot", [](ps_cuda_page_move &m) { m.n_kv = (1 << 30) + 1; });
    move("keeps below zero", I, "keeps", [](ps_cuda_page_move &m) { m.n_keep = -1; });
    move("keeps more than there are", I, "keeps", [](ps_cuda_page_move &m) { m.n_keep = 27; });
    move("no table", I, "no table", [](ps_cuda_page_move &m) { m.table = nullptr; });
    move("no list", I, "no table", [](ps_cuda_page_move &m) { m.keep = nullptr; });
    move("odd list", I, "no table", [](ps_cuda_page_move &m) { m.keep = odd<int32_t>(); });
    move("odd count", I, "no table", [](ps_cuda_page_move &m) { m.n_keep_dev = odd<int32_t>(); });
    move("short table", I, "its table", [](ps_cuda_page_move &m) { m.n_table = 1; });
    move("keeps nothing", 0, nullptr, [](ps_cuda_page_move &m) { m.n_keep = 0; m.table = nullptr; });
    expect("no moves", I, "no moves", [&](PsServeCall *c) { return ps_serve_paged_compact(c, &good, nullptr, 1); });
    expect("moves below zero", I, "no moves", [&](PsServeCall *c) { return ps_serve_paged_compact(c, &good, &some, -1); });

    // drafted tokens
    int32_t *ints = reinterpret_cast<int32_t *>(mem);
    const ps_cuda_sampler *set = reinterpret_cast<ps_cuda_sampler *>(mem);
    const int32_t three[2] = {3, 2}, zero[1] = {0}, wide[1] = {257};
    std::vector<int32_t> many(5000, 256);
    auto verify = [&](const char *name, int want, const char *text, const int32_t *nodes = nullptr, int n = 2, int64_t stride = 8, int64_t vocab = 8, int32_t *ids = nullptr, const float *lg = mem, const float *dl = nullptr,
                      const ps_cuda_sampler *ds = nullptr, const float *u = mem) {
        expect(name, want, text, [&](PsServeCall *c) { return ps_serve_verify(c, ids, ints, ints, nodes, n, ints, ints, lg, stride, vocab, set, u, dl, ds); });
    };
    verify("a call that is right asks for memory", PS_CUDA_ERR_OOM, nullptr, three, 2, 8, 8, ints);
    verify("no sequences", I, "no sequences");
    verify("sequences below zero", I, "no sequences", three, -1);
    verify("none", 0, nullptr, nullptr, 0);
    verify("no node", I, "nodes", zero, 1);
    verify("too many nodes", U, "nodes", wide, 1);
    verify("far too many nodes", U, "in one call", many.data(), 5000);
    verify("no vocabulary", I, "rows of", three, 2, 8, 0);
    verify("vocabulary above", I, "rows of", three, 2, 1 << 20, (1 << 18) + 1);
    verify("rows that overlap", I, "rows of", three, 2, 7, 8);
    verify("no ids", I, "null", three);
    verify("no logits", I, "null", three, 2, 8, 8, ints, nullptr);
    verify("no numbers", I, "null", three, 2, 8, 8, ints, mem, nullptr, nullptr, nullptr);
    verify("a draft without settings", I, "together", three, 2, 8, 8, ints, mem, mem);
    verify("settings without a draft", I, "together", three, 2, 8, 8, ints, mem, nullptr, set);
    verify("odd ids", I, "aligned", three, 2, 8, 8, odd<int32_t>());
    verify("odd logits", I, "aligned", three, 2, 8, 8, ints, odd<float>());
    printf(bad ? "%d wrong\n" : "all refused\n", bad);
    return bad != 0;
}
"""


def test_every_call_that_is_ruled_out_is_refused(tmp_path):
    lib = build.build()
    src, exe = tmp_path / "driver.cpp", tmp_path / "driver"
    src.write_text("#include <vector>\n" + DRIVER)
    cuda = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))
    cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-I" + ROOT, "-I" + os.path.join(cuda, "include"), str(src), lib, "-Wl,-rpath," + os.path.dirname(lib),
           "-L" + os.path.join(cuda, "lib64"), "-Wl,-rpath," + os.path.join(cuda, "lib64"), "-lcudart", "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_records_are_the_headers():
    """sizes and places of the fields, by the compiler"""
    import tempfile
    names = {"ps_cuda_paged_seq": capi.PAGED_SEQ, "ps_cuda_page_edit": capi.PAGE_EDIT, "ps_cuda_page_move": capi.PAGE_MOVE}
    lines = [f'printf("%zu {len(d)} %zu\\n", sizeof({n}), offsetof({n}, {d.names[-1]}));' for n, d in names.items()]
    lines.append('printf("%zu 0 %zu\\n", sizeof(ps_cuda_pages), offsetof(ps_cuda_pages, head_size));')
    with tempfile.TemporaryDirectory() as t:
        src = os.path.join(t, "r.cpp")
        with open(src, "w") as f:
            f.write('#include "include/ps_cuda.h"\n#include <cstdio>\n#include <cstddef>\nint main() {' + "".join(lines) + "}")
        subprocess.run([os.environ.get("CXX", "g++"), "-I" + ROOT, src, "-o", src + ".x"], check=True)
        got = [[int(x) for x in line.split()] for line in subprocess.run([src + ".x"], capture_output=True, text=True, check=True).stdout.splitlines()]
    want = [[d.itemsize, len(d), d.fields[d.names[-1]][1]] for d in names.values()]
    import ctypes
    assert got == want + [[ctypes.sizeof(capi.Pages), 0, capi.Pages.head_size.offset]]


class _NoDevice(capi.CudaBackend):
    def __init__(self):
        self.h, self.device, self.stream, self.L, self.calls = 1, 0, 0, type("L", (), {"__getattr__": lambda s, n: n})(), []

    def _in_turn(self, call, *args):
        self.calls.append((call, args))

    def close(self):
        pass


def test_arguments_that_python_refuses():
    import torch
    be = _NoDevice()
    cache = capi.PagedCache(be, 1, 4, 16, 2, 64, codes=4096, scales=8192, refs=12288)
    seqs = np.zeros(2, capi.PAGED_SEQ)
    seqs["n_kv"], seqs["n_tok"], seqs["n_table"] = 20, 3, 2
    for bad in (seqs.astype(capi.PAGED_SEQ)[::-1], seqs.tolist(), np.zeros(2, capi.CACHE)):
        for call in (lambda s: be.paged_store(cache, 0, 16, 16, s), lambda s: be.paged_load(cache, 0, 16, 16, s), lambda s: be.paged_attn(cache, 0, 16, 16, s, 4, 1.0)):
            with pytest.raises(capi.PsCudaError, match="PAGED_SEQ"):
                call(bad)
    with pytest.raises(capi.PsCudaError, match="PAGE_EDIT"):
        be.paged_edit(cache, seqs)
    with pytest.raises(capi.PsCudaError, match="PAGE_MOVE"):
        be.paged_compact(cache, seqs)
    host = torch.zeros(6, 128)
    with pytest.raises(capi.PsCudaError, match="memory of device"):
        be.paged_store(cache, 0, host, host, seqs)
    with pytest.raises(capi.PsCudaError, match="float32 or bfloat16"):
        be.paged_store(cache, 0, host.half(), host.half(), seqs)
    with pytest.raises(capi.PsCudaError, match="not of the type named"):
        be.paged_attn(cache, 0, host, host, seqs, 4, 1.0, io_type=capi.BF16)
    with pytest.raises(capi.PsCudaError, match="not a list"):
        be.paged_attn(cache, 0, 16, [1.0], seqs, 4, 1.0)
    for shape in ((0, 4, 16, 2, 64), (1, 0, 16, 2, 64), (1, 4, 24, 2, 64), (1, 4, 16, 0, 64), (1, 4, 16, 2, 0)):
        with pytest.raises(capi.PsCudaError, match="a paged cache of"):
            capi.PagedCache(be, *shape, codes=4096, scales=8192)
    with pytest.raises(capi.PsCudaError, match="verify: logits"):
        be.verify(16, 16, 16, [1, 2], 16, 16, host, 128, 16, 16)
    assert not be.calls
    be.paged_store(cache, 0, 16, 32, seqs, io_type=capi.BF16)
    be.paged_load(cache, 0, None, 32, seqs)
    be.paged_attn(cache, 0, 16, 16, seqs, 4, 0.5)
    be.verify(16, 16, 16, [1, 2], 16, 16, 16, 128, 16, 16)
    names = [n for n, _ in be.calls]
    assert names == ["ps_cuda_paged_store", "ps_cuda_paged_load", "ps_cuda_paged_attn", "ps_cuda_verify"]
    assert be.calls[0][1][2:5] == (16, 32, capi.BF16) and be.calls[1][1][2:5] == (None, 32, capi.F32)


def test_caches_that_are_not_this_devices_or_have_no_memory():
    be, other = _NoDevice(), _NoDevice()
    other.device = 1
    mine, theirs = (capi.PagedCache(b, 1, 4, 16, 2, 64, codes=4096, scales=8192, refs=12288) for b in (be, other))
    seqs = np.zeros(1, capi.PAGED_SEQ)
    calls = [lambda c: be.paged_store(c, 0, 16, 16, seqs), lambda c: be.paged_load(c, 0, 16, 16, seqs), lambda c: be.paged_attn(c, 0, 16, 16, seqs, 4, 1.0), lambda c: be.paged_edit(c, np.zeros(1, capi.PAGE_EDIT)),
             lambda c: be.paged_compact(c, np.zeros(1, capi.PAGE_MOVE))]
    for call in calls:
        for bad in (theirs, None, 4096, mine.pages):
            with pytest.raises(capi.PsCudaError, match="a PagedCache in the memory of device 0"):
                call(bad)
    for which in ("codes", "scales", "refs"):       # a buffer that was freed, by the cache or beside it
        gone = capi.DeviceBuffer.__new__(capi.DeviceBuffer)
        gone.be, gone.nbytes, gone.ptr = be, 1 << 20, 4096
        cache = capi.PagedCache(be, 1, 4, 16, 2, 64, **{**dict(codes=4096, scales=8192, refs=12288), which: gone})
        gone.ptr = None
        for call in calls:
            with pytest.raises(capi.PsCudaError, match="given back"):
                call(cache)
    assert not be.calls
    for call in calls:
        call(mine)
    assert len(be.calls) == 5
