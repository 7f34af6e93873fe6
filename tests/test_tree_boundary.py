"""CPU checks of the speculative-decoding entry points' refusals: every argument check of the C layer returns its code
and message before any HIP call (the addresses are never dereferenced), the op module rejects CPU tensors, and the
workspace queries answer without a GPU."""
import pytest
import torch

from runtime import ext

A = 0x10000000             # 16-byte aligned addresses, far apart
AT = [A + i * 0x10000000 for i in range(16)]


@pytest.fixture(scope="module")
def lib():
    return ext.open_library()


def refused(lib, rc, code, msg):
    assert rc == code and msg in lib.dk_last_error().decode(), (rc, lib.dk_last_error())


def call(lib, fn, base, kw):
    assert set(kw) <= set(base)
    a = dict(base, **kw)
    return getattr(lib, fn)(*a.values(), None)


QK = dict(qkv=AT[0], q_w=AT[1], k_w=AT[2], eps=1e-6, cos=AT[3], sin=AT[4], pos=AT[5], depth=AT[6], bt=AT[7], kc=AT[8],
          vc=AT[9], q_out=AT[10], q_stride=512, M=4, n_q=8, n_kv=2, head_dim=64, page=16, max_pos=64, n_pages=8, n_bt=8)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(qkv=None), 1, "null"), (dict(q_out=None), 1, "null"), (dict(cos=None), 1, "null"), (dict(bt=None), 1, "null"),
    (dict(q_w=None), 1, "together"), (dict(k_w=None), 1, "together"), (dict(head_dim=96), 3, "head_dim"),
    (dict(n_q=0), 3, "head counts"), (dict(n_kv=65536), 3, "head counts"), (dict(M=0), 3, "M must be"),
    (dict(M=(1 << 20) + 1), 3, "M must be"), (dict(page=12), 4, "power of two"), (dict(page=0), 4, "power of two"),
    (dict(max_pos=0), 3, "empty"), (dict(n_pages=0), 3, "empty"), (dict(n_bt=0), 3, "empty"),
    (dict(q_out=AT[10] + 8), 2, "16B aligned"), (dict(cos=AT[3] + 4), 2, "16B aligned"), (dict(q_w=AT[1] + 2), 2, "16B"),
    (dict(depth=AT[6] + 2), 2, "4B aligned"), (dict(pos=AT[5] + 1), 2, "4B aligned"), (dict(q_stride=504), 3, "q_stride"),
    (dict(q_stride=516), 3, "q_stride"), (dict(q_out=AT[0]), 4, "disjoint"), (dict(q_out=AT[0] + 1024, q_stride=768), 4, "disjoint")])
def test_qk_norm_rope_refusals(lib, kw, code, msg):
    refused(lib, call(lib, "dk_qk_norm_rope_append_rows", QK, kw), code, msg)


TREE = dict(q=AT[0], q_stride=1024, mask=AT[1], pos=AT[2], bt=AT[3], n_bt=8, kc=AT[4], vc=AT[5], n_pages=8, page=16, n_q=8,
            n_kv=2, head_dim=128, M=20, max_ctx=100, out=AT[6], ws=AT[7], ws_bytes=1 << 20)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(q=None), 1, "null"), (dict(out=None), 1, "null"), (dict(pos=None), 1, "null"), (dict(head_dim=32), 3, "head_dim"),
    (dict(M=0), 3, "M must be 1..1024"), (dict(M=1025), 3, "M must be 1..1024"), (dict(max_ctx=0), 4, "max_ctx"),
    (dict(max_ctx=(1 << 30) + 1), 4, "max_ctx must be 1..1073741824"),
    (dict(n_q=6), 3, "heads-per-group"), (dict(n_q=32), 3, "heads-per-group"), (dict(n_kv=0), 3, "heads-per-group"),
    (dict(n_kv=65536, n_q=65536), 3, "too many"), (dict(page=24), 4, "power of two"), (dict(n_bt=0), 3, "empty"),
    (dict(n_pages=0), 3, "empty"), (dict(q_stride=1020), 3, "q_stride"), (dict(q_stride=512), 3, "q_stride"),
    (dict(q=AT[0] + 8), 2, "16B"), (dict(out=AT[6] + 2), 2, "16B"), (dict(mask=AT[1] + 4), 2, "8B"),
    (dict(bt=AT[3] + 2), 2, "4B"), (dict(out=AT[0] + 64), 4, "overlap q"), (dict(out=AT[1] - 16), 4, "overlap q or mask"), (dict(ws=AT[7] + 8), 2, "workspace must be 16B")])
def test_attention_tree_refusals(lib, kw, code, msg):
    refused(lib, call(lib, "dk_attention_tree", TREE, kw), code, msg)


def test_attention_tree_workspace(lib):
    need = lib.dk_attention_tree_workspace_bytes
    assert need(0, 8, 2, 128, 100) == need(20, 6, 2, 128, 100) == need(20, 8, 2, 96, 100) == need(20, 8, 2, 128, 0) == 0
    assert need(1025, 8, 2, 128, 100) == 0
    big = need(64, 32, 8, 128, 1 << 20)
    assert big % 16 == 0
    if big:                          # a workspace that the call would use must overlap nothing
        kw = dict(M=64, n_q=32, n_kv=8, q_stride=4096, max_ctx=1 << 20, ws_bytes=big)
        for ws in (AT[0] + 160, AT[6] + 16, AT[1]):
            refused(lib, call(lib, "dk_attention_tree", TREE, dict(kw, ws=ws)), 4, "workspace must not overlap")


LP = dict(logits=AT[0], dtype=0, ld=1000, tokens=AT[1], logprobs=AT[2], entropy=AT[3], top_ids=AT[4], top=AT[5], M=4, V=1000,
          k=5, ws=AT[6], ws_bytes=1 << 20)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(logits=None), 1, "null"), (dict(dtype=3), 4, "dtype"), (dict(dtype=-1), 4, "dtype"), (dict(M=0), 3, "M must"),
    (dict(V=0), 3, "V must"), (dict(V=(1 << 24) + 1), 3, "V must"), (dict(k=33), 3, "k must"), (dict(k=-1), 3, "k must"),
    (dict(V=4, k=5), 3, "k must"), (dict(tokens=None), 1, "together"), (dict(logprobs=None), 1, "together"),
    (dict(top_ids=None), 1, "belong to k > 0"), (dict(k=0), 1, "belong to k > 0"),
    (dict(k=0, top_ids=None, top=None, tokens=None, logprobs=None, entropy=None), 1, "no output"),
    (dict(ld=999), 3, "row stride"), (dict(logits=AT[0] + 1), 2, "aligned"), (dict(dtype=2, logits=AT[0] + 2), 2, "aligned"),
    (dict(tokens=AT[1] + 4), 2, "8B"), (dict(entropy=AT[3] + 2), 2, "4B"), (dict(logprobs=AT[0] + 16), 4, "overlap"),
    (dict(entropy=AT[2] + 8), 4, "overlap"), (dict(top=AT[4] + 16), 4, "overlap"), (dict(logprobs=AT[1]), 4, "overlap"),
    (dict(ws=AT[6] + 4), 2, "workspace must be 16B")])
def test_token_logprobs_refusals(lib, kw, code, msg):
    refused(lib, call(lib, "dk_token_logprobs", LP, kw), code, msg)


def test_token_logprobs_workspace(lib):
    need = lib.dk_token_logprobs_workspace_bytes
    assert need(0, 1000, 5, 0) == need(1, 1000, 33, 0) == need(1, 1000, 5, 3) == need(1, 4, 5, 0) == 0
    n = need(1, 128256, 5, 0)
    if n:
        kw = dict(M=1, V=128256, ld=128256, ws_bytes=n)
        for ws in (AT[0], AT[1], AT[3]):
            refused(lib, call(lib, "dk_token_logprobs", LP, dict(kw, ws=ws)), 4, "workspace must overlap neither")


ACC = dict(tokens=AT[0], parents=AT[1], picks=AT[2], stride=1, M=10, pos=AT[3], bt=AT[4], n_bt=8, kv=AT[5], n_caches=4,
           n_pages=8, n_kv=2, page=16, head_dim=64, path=AT[6], count=AT[7], tok=AT[8])


@pytest.mark.parametrize("kw,code,msg", [
    (dict(tokens=None), 1, "null"), (dict(path=None), 1, "null"), (dict(pos=None), 1, "null"), (dict(M=0), 3, "M must be"),
    (dict(M=1025), 3, "M must be"), (dict(stride=0), 3, "picks_stride"), (dict(kv=None), 3, "both be given"),
    (dict(n_caches=0), 3, "both be given"), (dict(n_caches=-1, kv=None), 3, "both be given"), (dict(head_dim=72), 3, "head_dim"),
    (dict(n_kv=0), 3, "head count"), (dict(page=10), 4, "power of two"), (dict(n_pages=0), 3, "empty"),
    (dict(kv=AT[5] + 8), 2, "kv must be 16B"), (dict(picks=AT[2] + 4), 2, "8B"), (dict(path=AT[6] + 2), 2, "4B"),
    (dict(tok=AT[0] + 8), 4, "overlap"), (dict(path=AT[1] + 16), 4, "overlap"), (dict(count=AT[3]), 4, "overlap"),
    (dict(count=AT[6] + 36), 4, "overlap"), (dict(tok=AT[2] + 80, stride=2), 4, "overlap")])
def test_tree_accept_refusals(lib, kw, code, msg):
    refused(lib, call(lib, "dk_tree_accept", ACC, kw), code, msg)


def test_workspace_queries_refuse_sizes_past_32_bits(lib):
    K = ext.DecodeKernels(lib)
    for sizes in ((20, 32, 8, 128, (1 << 32) + 9000), ((1 << 32) + 20, 32, 8, 128, 9000)):
        with pytest.raises(RuntimeError, match="32 bits"):
            K.attention_tree_workspace_bytes(*sizes)
    for sizes in ((1, (1 << 32) + 128256, 5), ((1 << 32) + 1, 128256, 5), (1, 128256, 5 - (1 << 32))):
        with pytest.raises(RuntimeError, match="32 bits"):
            K.token_logprobs_workspace_bytes(*sizes)


def test_op_module_rejects_cpu_tensors(lib):
    K = ext.DecodeKernels(lib)
    h = lambda *s: torch.zeros(*s, dtype=torch.half)
    kc, bt, pos = h(4, 2, 16, 64), torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    ids, f = torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.qk_norm_rope_append_rows(h(3, 384), None, None, 0.0, torch.zeros(8, 32), torch.zeros(8, 32), pos, None, bt, kc, kc, 2, 2)
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.attention_tree(h(3, 2, 64), None, pos, bt, kc, kc, 10, h(3, 128))
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.token_logprobs(h(3, 100), ids, f)
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.tree_accept(ids, ids.int(), ids, pos, bt, kc, ids.int(), pos.clone(), ids[:1])
    with pytest.raises(RuntimeError, match="fp16, bf16 or fp32"):
        K.token_logprobs_workspace_bytes(1, 10, 1, torch.float64)
