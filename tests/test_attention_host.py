"""The attention operators' C surface without a GPU: struct layouts, constants, and refusals of a missing context."""
import ctypes as C
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "mrl_kv.h")).read()


def fields(name):
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1), flags=re.S)
    out = []
    for decl in body.split(";"):
        decl = " ".join(decl.split())
        if not decl:
            continue
        kind = "pointer" if "*" in decl else decl.split()[0]
        out += [(n.replace("*", "").split()[-1], kind) for n in decl.split(",")]
    return out


def test_structs_match_the_header():
    from mrl_b200._capi import AttnC, KvCacheC

    kinds = {"pointer": C.c_void_p, "int64_t": C.c_int64, "uint32_t": C.c_uint32, "float": C.c_float}
    for name, struct in (("mrl_kv_cache", KvCacheC), ("mrl_attn", AttnC)):
        assert [(n, kinds[k]) for n, k in fields(name)] == list(struct._fields_)


def test_constants_match_the_header():
    from mrl_b200 import attention as A

    value = lambda n: int(re.search(r"#define %s (\d+)u" % n, HEADER).group(1))  # noqa: E731
    assert A.PAGE_TOKENS == value("MRL_KV_PAGE")
    assert (A.KV_NO_PAGES, A.KV_ROW_FULL, A.KV_BAD_INDEX, A.KV_NONFINITE, A.KV_TIMEOUT) == tuple(
        value("MRL_KV_" + n) for n in ("NO_PAGES", "ROW_FULL", "BAD_INDEX", "NONFINITE", "TIMEOUT"))


def test_calls_without_a_context_are_refused():
    from mrl_b200 import _capi

    lib = _capi.load()
    for name, (_, args) in _capi.SIGNATURES.items():
        if name.startswith("mrl_kv_") or name in ("mrl_window_attention", "mrl_ctx_join"):
            assert getattr(lib, name)(*[None if a is C.c_void_p else 0 for a in args]) == _capi.MRL_ERR_INVALID, name


def test_cases_state_their_work():
    """perf/operators.py lists distinct cases with positive work, over a range of at least 16, without a GPU."""
    import importlib.util
    import random

    spec = importlib.util.spec_from_file_location("operators_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    cases = m.listed()
    assert len({c["name"] for c in cases}) == len(cases)
    work = [max(m.work(c)["bytes"], m.work(c)["flops"] / 50) for c in cases]
    assert min(work) > 0 and max(work) >= 16 * min(work)
    rng = random.Random(1)
    for _ in range(40):
        c = m.draw(rng)
        assert m.work(c)["bytes"] > 0 and max(m.work(c)["bytes"], m.work(c)["flops"] / 50) <= max(work)
