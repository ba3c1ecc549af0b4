"""The serving operators' host side (serve.c) without a GPU: the file is
compiled against stand-ins of hip_backend.h's calls that write down what would
be launched.

  - every documented limit of trlm_serve.h is refused with -1, a message and
    nothing launched, and the values next to it are taken;
  - a call with nothing to do launches nothing and returns 0;
  - the grids cover every row, and the workspace query agrees with what the
    call asks for;
  - the header's functions are exported by the built library, its structures
    are the binding's, and the code object holds every kernel of the file;
  - the kernels' argument blocks are the host's structures."""
import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "turkce-llm_amd", "csrc")
ROCM_INC = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")
needs_hip = pytest.mark.skipif(not os.path.exists(os.path.join(ROCM_INC, "hip", "hip_runtime_api.h")),
                               reason="HIP headers not present")

STUBS = r"""
#include "serve.c"
static int cur_device;
char launched[4096];
hipFunction_t hip_get_kernel(HipCtx* c, const char* name) { (void)c; return (hipFunction_t)strdup(name); }
void hip_launch(hipFunction_t f, u32 gx, u32 gy, u32 gz, u32 bx, u32 by, u32 bz, u32 shared, void** args) {
    (void)gz; (void)by; (void)bz; (void)shared; (void)args;
    const size_t n = strlen(launched);
    snprintf(launched + n, sizeof(launched) - n, "%s %u %u %u;", (const char*)f, gx, gy, bx);
}
hipError_t hipGetDevice(int* d) { *d = cur_device; return hipSuccess; }
void set_device(int d) { cur_device = d; }
void clear_launched(void) { launched[0] = 0; }
const char* get_launched(void) { return launched; }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory, trlm):
    """serve.c over the stand-ins, as a library of its own."""
    d = tmp_path_factory.mktemp("serve")
    src, so = d / "serve_stub.c", d / "libserve_stub.so"
    src.write_text(STUBS)
    subprocess.run(["gcc", "-std=c11", "-O1", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-Wall", "-D_DEFAULT_SOURCE", "-D__HIP_PLATFORM_AMD__",
                    "-I" + CSRC, "-I" + os.path.join(ROOT, "include"), "-I" + ROCM_INC, str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    cache, seqs = C.POINTER(trlm.KvCache), C.POINTER(trlm.KvSeqs)
    for name, res, args in [
            ("trlm_serve_create", C.c_void_p, [C.POINTER(trlm.HipCtx)]),
            ("trlm_kv_append", C.c_int32, [C.c_void_p, cache, seqs, C.POINTER(trlm.KvRows)]),
            ("trlm_kv_read", C.c_int32, [C.c_void_p, cache, seqs, C.c_void_p, C.c_void_p, C.c_uint32]),
            ("trlm_attn_paged_workspace", C.c_uint64, [cache, seqs, C.c_uint32]),
            ("trlm_attn_paged", C.c_int32, [C.c_void_p, cache, seqs, C.c_void_p, C.c_uint32, C.c_uint32, C.c_float,
                                            C.c_void_p, C.c_uint32, C.c_void_p, C.c_uint64]),
            ("trlm_logits_rules", C.c_int32, [C.c_void_p, C.POINTER(trlm.LogitsRules)]),
            ("get_launched", C.c_char_p, []), ("clear_launched", None, []), ("set_device", None, [C.c_int32])]:
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    ctx = trlm.HipCtx()
    lib.ctx = ctx
    lib.e = lib.trlm_serve_create(C.byref(ctx))
    lib.clear_launched()
    return lib


def cache(trlm, **k):
    a = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, type=0, num_pages=10, page_size=64, kv_heads=2,
             head_dim=64)
    return trlm.KvCache(**(a | k))


def seqs(trlm, **k):
    a = dict(n=3, rows=8, q_start=0x1000, kv_len=0x2000, pages=0x3000, max_pages=4, max_q=5, max_kv=200)
    return trlm.KvSeqs(**(a | k))


def rows(trlm, **k):
    a = dict(q=0x50000, k=0x60000, v=0x70000, ldq=512, ldk=512, ldv=512, q_out=0x80000, ldqo=512, heads=4, cos_t=0x1000,
             sin_t=0x2000, max_pos=256, rot_dim=64, rot_half=0)
    return trlm.KvRows(**(a | k))


def rules(trlm, **k):
    a = dict(logits=0x10000, out=0x20000, rows=4, vocab=1000, ld=1000, ld_out=1000, history=0x30000, hist_len=0x40000,
             gen_start=None, ld_hist=50, repetition=0x50000, frequency=None, presence=None, bias_ids=0x60000,
             bias=0x61000, n_bias=0x62000, ld_bias=8, mask=0x70000, ld_mask=32)
    return trlm.LogitsRules(**(a | k))


def outcome(host, call, capfd):
    """(return value, launches, message) of a call."""
    host.clear_launched()
    rc = call()
    return rc, host.get_launched().decode(), capfd.readouterr().err


def refused(host, call, capfd, op, handle=False):
    rc, launched, err = outcome(host, call, capfd)
    assert rc == -1 and launched == "" and err.startswith(op + ": refused, nothing launched: "), (rc, launched, err)
    assert ("handle" in err) == handle, err


def taken(host, call, capfd):
    rc, launched, err = outcome(host, call, capfd)
    assert rc == 0 and launched and not err, (rc, launched, err)
    return launched


BAD_CACHE = [dict(k=None), dict(v=None), dict(k=0x10008), dict(v=0x20004), dict(type=3), dict(num_pages=0),
             dict(num_pages=2 ** 31), dict(page_size=8), dict(page_size=48), dict(page_size=0), dict(page_size=131072),
             dict(kv_heads=0), dict(kv_heads=1025), dict(head_dim=0), dict(head_dim=48), dict(head_dim=256),
             dict(type=2, k_scale=None), dict(type=2, v_scale=0x40004)]
BAD_SEQS = [dict(n=4097), dict(rows=2 ** 24), dict(max_pages=0), dict(max_pages=2 ** 25), dict(q_start=None),
            dict(kv_len=None), dict(pages=None), dict(pages=0x3002)]
BAD_ROWS = [dict(k=None), dict(v=None), dict(k=0x60004), dict(ldk=510), dict(ldk=124), dict(ldv=100), dict(q=None),
            dict(q_out=None), dict(heads=0), dict(heads=1025), dict(q=0x50004), dict(ldq=252), dict(ldqo=514),
            dict(ldqo=252), dict(q_out=0x50000, ldqo=516), dict(rot_dim=4), dict(rot_dim=72), dict(cos_t=None),
            dict(sin_t=0x2004), dict(max_pos=0)]
BAD_RULES = [dict(logits=None), dict(out=None), dict(logits=0x10002), dict(vocab=0), dict(vocab=2 ** 30 + 1),
             dict(ld=999), dict(ld_out=999), dict(rows=65536), dict(out=0x10000, ld_out=1004), dict(hist_len=None),
             dict(ld_hist=0), dict(bias=None), dict(n_bias=None), dict(ld_bias=0), dict(ld_mask=31), dict(mask=0x70001)]


@needs_hip
@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_caches_out_of_range(host, trlm, capfd, bad):
    c, s = cache(trlm, **bad), seqs(trlm)
    refused(host, lambda: host.trlm_kv_append(host.e, c, s, rows(trlm)), capfd, "trlm_kv_append")
    refused(host, lambda: host.trlm_kv_read(host.e, c, s, 0x1000, 0x2000, 128), capfd, "trlm_kv_read")
    refused(host, lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 512, 4, 0.125, 0x2000, 512, 0x3000, 2 ** 40), capfd,
            "trlm_attn_paged")
    assert host.trlm_attn_paged_workspace(c, s, 4) == 0


@needs_hip
@pytest.mark.parametrize("bad", BAD_SEQS, ids=str)
def test_sequences_out_of_range(host, trlm, capfd, bad):
    c, s = cache(trlm), seqs(trlm, **bad)
    refused(host, lambda: host.trlm_kv_append(host.e, c, s, rows(trlm)), capfd, "trlm_kv_append")
    refused(host, lambda: host.trlm_kv_read(host.e, c, s, 0x1000, 0x2000, 128), capfd, "trlm_kv_read")
    refused(host, lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 512, 4, 0.125, 0x2000, 512, 0x3000, 2 ** 40), capfd,
            "trlm_attn_paged")


@needs_hip
@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_rows_out_of_range(host, trlm, capfd, bad):
    refused(host, lambda: host.trlm_kv_append(host.e, cache(trlm), seqs(trlm), rows(trlm, **bad)), capfd, "trlm_kv_append")


@needs_hip
@pytest.mark.parametrize("bad", BAD_RULES, ids=str)
def test_rules_out_of_range(host, trlm, capfd, bad):
    refused(host, lambda: host.trlm_logits_rules(host.e, rules(trlm, **bad)), capfd, "trlm_logits_rules")


@needs_hip
def test_other_arguments_out_of_range(host, trlm, capfd):
    c, s = cache(trlm), seqs(trlm)
    for a in ((None, 0x2000, 128), (0x1000, None, 128), (0x1004, 0x2000, 128), (0x1000, 0x2000, 126), (0x1000, 0x2000, 124)):
        refused(host, lambda: host.trlm_kv_read(host.e, c, s, *a), capfd, "trlm_kv_read")
    assert host.trlm_attn_paged_workspace(c, s, 4) == 0  # a short context is not split: no workspace is asked for
    taken(host, lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 512, 4, 0.125, 0x2000, 512, None, 0), capfd)
    s = seqs(trlm, max_pages=40, max_kv=2000)
    ws = host.trlm_attn_paged_workspace(c, s, 4)
    assert ws > 0
    good = (0x1000, 512, 4, 0.125, 0x2000, 512, 0x3000, ws)
    taken(host, lambda: host.trlm_attn_paged(host.e, c, s, *good), capfd)
    for at, v in ((0, None), (0, 0x1004), (1, 252), (1, 510), (2, 0), (2, 3), (2, 1026), (4, None), (5, 252), (6, 0x3008),
                  (6, None), (7, ws - 1)):
        a = list(good)
        a[at] = v
        refused(host, lambda: host.trlm_attn_paged(host.e, c, s, *a), capfd, "trlm_attn_paged")
    s = seqs(trlm, rows=2 ** 21, max_q=1, max_kv=64)
    c = cache(trlm, kv_heads=1, head_dim=16)
    refused(host, lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 16384, 1024, 0.125, 0x2000, 16384, 0x3000, 2 ** 62),
            capfd, "trlm_attn_paged")
    # more threads than a launch holds: 2^24 workgroups of 256, 2^23 of 512, 2^24 of joins
    c = cache(trlm, kv_heads=1024, head_dim=16, num_pages=1000)
    for heads, k in ((1024, dict(n=4096, rows=4096 * 64, max_q=64)), (1024, dict(n=2048, rows=2 ** 20, max_q=1024))):
        s = seqs(trlm, max_kv=64, **k)
        refused(host, lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 16384, heads, 0.125, 0x2000, 16384, 0x3000, 2 ** 62),
                capfd, "trlm_attn_paged")
    c, s = cache(trlm, kv_heads=1, head_dim=128), seqs(trlm, n=1, rows=2 ** 20, max_q=1, max_kv=2 ** 16,
                                                          max_pages=2 ** 10)
    refused(host, lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 2 ** 17, 1024, 0.125, 0x2000, 2 ** 17, 0x3000, 2 ** 62),
            capfd, "trlm_attn_paged")


@needs_hip
def test_another_device_or_no_handle(host, trlm, capfd):
    calls = {"trlm_kv_append": lambda e: host.trlm_kv_append(e, cache(trlm), seqs(trlm), rows(trlm)),
             "trlm_kv_read": lambda e: host.trlm_kv_read(e, cache(trlm), seqs(trlm), 0x1000, 0x2000, 128),
             "trlm_attn_paged": lambda e: host.trlm_attn_paged(e, cache(trlm), seqs(trlm), 0x1000, 512, 4, 1.0, 0x2000, 512,
                                                               0x3000, 2 ** 40),
             "trlm_logits_rules": lambda e: host.trlm_logits_rules(e, rules(trlm))}
    for op, call in calls.items():
        host.set_device(1)
        refused(host, lambda: call(host.e), capfd, op, handle=True)
        host.set_device(0)
        refused(host, lambda: call(None), capfd, op, handle=True)
        taken(host, lambda: call(host.e), capfd)


@needs_hip
def test_nothing_to_do(host, trlm, capfd):
    c = cache(trlm)
    for s in (seqs(trlm, n=0), seqs(trlm, rows=0)):
        for call in (lambda: host.trlm_kv_append(host.e, c, s, rows(trlm)),
                     lambda: host.trlm_kv_read(host.e, c, s, 0x1000, 0x2000, 128),
                     lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 512, 4, 1.0, 0x2000, 512, None, 0)):
            assert outcome(host, call, capfd) == (0, "", "")
    s = seqs(trlm, max_q=0)
    assert outcome(host, lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 512, 4, 1.0, 0x2000, 512, None, 0),
                   capfd) == (0, "", "")
    assert outcome(host, lambda: host.trlm_logits_rules(host.e, rules(trlm, rows=0)), capfd) == (0, "", "")


@needs_hip
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("n_rows", [1, 15, 17, 2000, 70001])
def test_cache_grids_cover_the_rows(host, trlm, capfd, hd, n_rows):
    c, s = cache(trlm, head_dim=hd, type=1), seqs(trlm, rows=n_rows)
    for text, heads in ((taken(host, lambda: host.trlm_kv_append(host.e, c, s, rows(trlm, rot_dim=16)), capfd), 8),
                        (taken(host, lambda: host.trlm_kv_read(host.e, c, s, 0x1000, 0x2000, 256), capfd), 4)):
        name, gx, gy, bx = text.rstrip(";").split()
        per, wide = 1024 // hd, 4 if re.match(r"k_kv_\w+4_hd", name) else 1
        assert name.endswith("_hd%d_bf16" % hd) and int(bx) == 256
        assert int(gy) == -(-heads // wide) and (int(gx) - 1) * per < n_rows <= int(gx) * per


@needs_hip
@pytest.mark.parametrize("max_kv", [0, 1, 128, 129, 5000, 10 ** 9])
@pytest.mark.parametrize("n,n_rows,max_q", [(1, 1, 1), (64, 64, 1), (3, 8, 5), (2, 700, 10 ** 6)])
def test_attention_splits_cover_the_context(host, trlm, capfd, max_kv, n, n_rows, max_q):
    c = cache(trlm, page_size=64)
    s = seqs(trlm, n=n, rows=n_rows, max_q=max_q, max_kv=max_kv, max_pages=100)
    ws = host.trlm_attn_paged_workspace(c, s, 6)
    text = taken(host, lambda: host.trlm_attn_paged(host.e, c, s, 0x1000, 512, 6, 1.0, 0x2000, 512, 0x3000, ws), capfd)
    parts = [p.split() for p in text.rstrip(";").split(";")]
    joins = [p for p in parts if p[0] in ("k_paged_attn_join_hd64", "k_paged_attn_join_long_hd64")]
    per = 4 if joins and "long" in joins[0][0] else 16
    assert bool(joins) == (ws > 0)
    if joins:
        splits = ws // (n_rows * 6 * 66 * 4)
        assert ws == n_rows * 6 * 66 * 4 * splits and splits > 1
        assert (int(joins[0][1]) - 1) * per < n_rows * 6 <= int(joins[0][1]) * per
        assert max(int(p[2]) for p in parts) == splits


def test_header_and_binding_agree(trlm, tmp_path):
    with open(os.path.join(ROOT, "include", "trlm_serve.h")) as fh:
        text = re.sub(r"/\*.*?\*/", "", fh.read(), flags=re.S)
    _, hip = trlm.libs()
    names = set(re.findall(r"^(?:i32|u32|u64|f32|void|[A-Z]\w+\*) ((?:trlm|gpu)_\w+)\(", text, re.M))
    assert {"gpu_paged_create", "gpu_paged_extend", "gpu_paged_rules", "gpu_paged_read", "trlm_serve_create",
            "trlm_serve_destroy", "trlm_kv_append", "trlm_kv_read", "trlm_attn_paged", "trlm_attn_paged_workspace",
            "trlm_logits_rules"} <= names
    for n in names:
        assert hasattr(hip, n), n
    if not os.path.exists(os.path.join(ROCM_INC, "hip", "hip_runtime_api.h")):
        return
    mirrors = {"TrlmKvCache": trlm.KvCache, "TrlmKvSeqs": trlm.KvSeqs, "TrlmKvRows": trlm.KvRows,
               "TrlmLogitsRules": trlm.LogitsRules, "TrlmTokenRules": trlm.TokenRules}
    out = []
    for s, m in mirrors.items():
        out += ['printf("%%zu ", sizeof(%s));' % s] + ['printf("%%zu ", offsetof(%s, %s));' % (s, f) for f, _ in m._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "trlm_serve.h"\nint main(void) { %s return 0; }\n' %
                   "".join(out))
    subprocess.run(["gcc", "-std=c11", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(ROOT, "include"), "-I" + ROCM_INC,
                    str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for m in mirrors.values():
        want += [C.sizeof(m)] + [getattr(m, f).offset for f, _ in m._fields_]
    assert got == want


def kernel_names():
    names = {"k_%s_hd%d_%s" % (k, hd, t) for k in ("kv_append", "kv_append4", "kv_read", "kv_read4", "paged_attn_few",
                                               "paged_attn_tile", "paged_attn_mixed")
             for hd in (16, 32, 64, 128) for t in ("f32", "bf16", "i8")}
    names |= {"k_paged_attn_join%s_hd%d" % (k, hd) for k in ("", "_long") for hd in (16, 32, 64, 128)}
    return names | {"k_logits_rules_%d%s" % (w, u) for w in (1024, 4096) for u in ("", "_u")}


def test_code_object_has_the_kernels(trlm):
    with open(trlm.KERNELS, "rb") as fh:
        blob = fh.read()
    for n in sorted(kernel_names()):
        assert n.encode() + b"\0" in blob, n


LLVM = "/opt/rocm/llvm/bin"


@pytest.mark.skipif(not os.path.exists(os.path.join(LLVM, "llvm-readobj")), reason="ROCm LLVM tools not present")
def test_argument_blocks_match_the_host(trlm, tmp_path):
    """As test_abi.py does for the other kernels: one by-value argument of exactly the host structure's size; and no
    kernel spills to scratch memory."""
    import yaml
    src, exe = tmp_path / "kp.c", tmp_path / "kp"
    src.write_text('#include <stdio.h>\n#include "kernel_params.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", '
                   'sizeof(KvAppendParams), sizeof(KvReadParams), sizeof(PagedAttnParams), sizeof(RulesParams)); return 0; }\n')
    subprocess.run(["gcc", "-std=c11", "-I" + CSRC, str(src), "-o", str(exe)], check=True)
    sizes = dict(zip(("k_kv_append", "k_kv_read", "k_paged_attn", "k_logits_rules"), map(int, subprocess.run(
        [str(exe)], check=True, capture_output=True, text=True).stdout.split())))
    co = tmp_path / "k.co"
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--unbundle", "--type=o", "--input=" + trlm.KERNELS,
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--output=" + str(co)], check=True)
    notes = subprocess.run([os.path.join(LLVM, "llvm-readobj"), "--notes", str(co)], check=True, capture_output=True,
                           text=True).stdout
    a = notes.index("---")
    found = {k[".name"]: k for k in yaml.safe_load(notes[a:notes.index("\n...", a)])["amdhsa.kernels"]}
    for n in kernel_names():
        explicit = [x for x in found[n][".args"] if not x[".value_kind"].startswith("hidden_")]
        want = next(v for k, v in sizes.items() if n.startswith(k))
        assert len(explicit) == 1 and explicit[0][".value_kind"] == "by_value" and explicit[0][".size"] == want, n
        # (seven registers of the 128-wide tile forms' rare path)
        most = 32 if re.match(r"k_paged_attn_tile_hd128_(bf16|i8)", n) else 0
        most = 160 if "k_paged_attn_mixed_hd128" in n else most      # (looks its tiles up, in turns)
        assert found[n][".private_segment_fixed_size"] <= most, (n, "spills")
