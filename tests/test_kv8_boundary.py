"""CPU checks of the refusals of the 8-bit cache and of windowed attention: every argument check of the C layer returns its
code and message before any HIP call (the addresses are never dereferenced), the op module rejects CPU tensors and wrong
shapes, and the workspace query answers without a GPU."""
import pytest
import torch

from runtime import ext

A = 0x10000000
AT = [A + i * 0x10000000 for i in range(16)]


@pytest.fixture(scope="module")
def lib():
    return ext.open_library()


def refused(lib, fn, base, kw, code, msg):
    assert set(kw) <= set(base)
    rc = getattr(lib, fn)(*dict(base, **kw).values(), None)
    assert rc == code and msg in lib.dk_last_error().decode(), (rc, lib.dk_last_error())


APP = dict(qkv=AT[0], cos=AT[1], sin=AT[2], pos=AT[3], bt=AT[4], kc=AT[5], vc=AT[6], ks=AT[7], vs=AT[8], cache=1,
           q_out=AT[9], q_stride=512, M=4, n_q=8, n_kv=2, head_dim=64, page=16, max_pos=64, n_pages=8, n_bt=8)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(qkv=None), 1, "null"), (dict(ks=None), 1, "null"), (dict(vc=None), 1, "null"), (dict(q_out=None), 1, "null"),
    (dict(cos=None), 1, "together"), (dict(sin=None), 1, "together"), (dict(cache=0), 4, "int8 or e4m3"),
    (dict(cache=3), 4, "int8 or e4m3"), (dict(head_dim=96), 3, "head_dim"), (dict(n_kv=0), 3, "kv head count"),
    (dict(n_q=0), 3, "query head count"), (dict(n_q=65536), 3, "query head count"), (dict(page=8), 4, "power of two >= 16"),
    (dict(page=48), 4, "power of two >= 16"), (dict(n_pages=0), 3, "empty"), (dict(n_bt=0), 3, "empty"),
    (dict(M=0), 3, "M must be"), (dict(M=(1 << 20) + 1), 3, "M must be"), (dict(max_pos=0), 3, "empty rope"),
    (dict(qkv=AT[0] + 8), 2, "16B"), (dict(kc=AT[5] + 8), 2, "16B"), (dict(sin=AT[2] + 4), 2, "16B"),
    (dict(ks=AT[7] + 2), 2, "4B"), (dict(pos=AT[3] + 1), 2, "4B"), (dict(q_stride=504), 3, "q_stride"),
    (dict(q_stride=516), 3, "q_stride"), (dict(q_out=AT[0]), 4, "disjoint"),
    (dict(q_out=AT[0] + 1024, q_stride=768), 4, "disjoint"),
    (dict(M=1 << 20, n_kv=512, n_q=512, q_stride=512 * 64), 3, "too many rows")])
def test_kv8_append_refusals(lib, kw, code, msg):
    refused(lib, "dk_kv8_append_rows", APP, kw, code, msg)


READ = dict(bt=AT[0], n_bt=8, kc=AT[1], vc=AT[2], ks=AT[3], vs=AT[4], cache=2, n_pages=8, page=32, n_kv=2, head_dim=128,
            start=5, n=100, k_out=AT[5], v_out=AT[6])


@pytest.mark.parametrize("kw,code,msg", [
    (dict(bt=None), 1, "null"), (dict(vs=None), 1, "null"), (dict(k_out=None), 1, "null"), (dict(cache=0), 4, "int8 or e4m3"),
    (dict(head_dim=32), 3, "head_dim"), (dict(n_kv=65536), 3, "kv head count"), (dict(page=4), 4, "power of two >= 16"),
    (dict(n_bt=0), 3, "empty"), (dict(start=-1), 3, "range"), (dict(n=0), 3, "range"), (dict(n=1 << 30), 3, "range"),
    (dict(n=1 << 29, n_kv=8), 3, "too many"), (dict(kc=AT[1] + 8), 2, "16B"), (dict(v_out=AT[6] + 2), 2, "16B"),
    (dict(vs=AT[4] + 2), 2, "4B"), (dict(v_out=AT[5] + 160), 4, "overlap")])
def test_kv8_read_refusals(lib, kw, code, msg):
    refused(lib, "dk_kv8_read", READ, kw, code, msg)


WIN = dict(q=AT[0], q_stride=1024, pos=AT[1], bt=AT[2], n_bt=8, kc=AT[3], vc=AT[4], ks=AT[5], vs=AT[6], cache=2, n_pages=8,
           page=16, n_q=8, n_kv=2, head_dim=128, M=20, max_ctx=100, window=0, sinks=0, out=AT[7], ws=AT[8], ws_bytes=1 << 20)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(q=None), 1, "null"), (dict(out=None), 1, "null"), (dict(bt=None), 1, "null"), (dict(cache=3), 4, "cache must be"),
    (dict(cache=-1), 4, "cache must be"), (dict(ks=None), 1, "scales belong"), (dict(vs=None), 1, "scales belong"),
    (dict(cache=0), 1, "scales belong"), (dict(head_dim=96), 3, "head_dim"), (dict(M=0), 3, "M must be"),
    (dict(M=(1 << 20) + 1), 3, "M must be"), (dict(max_ctx=0), 4, "max_ctx"), (dict(max_ctx=(1 << 30) + 1), 4, "max_ctx"),
    (dict(window=-1), 4, "window and sinks"), (dict(sinks=-1), 4, "window and sinks"),
    (dict(window=(1 << 30) + 1), 4, "window and sinks"), (dict(n_q=6), 3, "heads-per-group"),
    (dict(n_q=32), 3, "heads-per-group"), (dict(n_kv=0), 3, "heads-per-group"), (dict(page=24), 4, "power of two"),
    (dict(page=8), 4, "16 tokens or more"), (dict(n_pages=0), 3, "empty"), (dict(n_bt=0), 3, "empty"),
    (dict(q_stride=1020), 3, "q_stride"), (dict(q_stride=512), 3, "q_stride"), (dict(q=AT[0] + 8), 2, "16B"),
    (dict(out=AT[7] + 2), 2, "16B"), (dict(vs=AT[6] + 2), 2, "4B"), (dict(out=AT[0] + 64), 4, "overlap q"),
    (dict(M=1 << 20, n_q=64, n_kv=8, q_stride=8192), 3, "too many rows"), (dict(ws=AT[8] + 8), 2, "workspace must be 16B")])
def test_attention_window_refusals(lib, kw, code, msg):
    refused(lib, "dk_attention_window", WIN, kw, code, msg)


DEC = dict(qkv=AT[0], cos=AT[1], sin=AT[2], max_pos=64, pos=AT[3], bt=AT[4], n_bt=8, kc=AT[5], vc=AT[6], ks=AT[7], vs=AT[8],
           cache=1, n_pages=8, page=16, n_q=8, n_kv=2, head_dim=64, max_ctx=64, window=0, sinks=0, out=AT[9], ws=None,
           ws_bytes=0)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(qkv=None), 1, "null"), (dict(cos=None), 1, "null"), (dict(sin=None), 1, "null"), (dict(ks=None), 1, "null"),
    (dict(out=None), 1, "null"), (dict(cache=0), 4, "int8 or e4m3"), (dict(head_dim=96), 3, "head_dim"),
    (dict(n_kv=0), 3, "kv head count"), (dict(page=8), 4, "power of two >= 16"), (dict(n_pages=0), 3, "empty"),
    (dict(max_pos=0), 3, "empty rope"), (dict(max_ctx=0), 4, "max_ctx"), (dict(max_ctx=(1 << 30) + 1), 4, "max_ctx"),
    (dict(window=-1), 4, "window and sinks"), (dict(sinks=(1 << 30) + 1), 4, "window and sinks"),
    (dict(n_q=6), 3, "heads-per-group"), (dict(n_q=32), 3, "heads-per-group"), (dict(qkv=AT[0] + 8), 2, "16B"),
    (dict(cos=AT[1] + 4), 2, "16B"), (dict(out=AT[9] + 2), 2, "16B"), (dict(bt=AT[4] + 2), 2, "4B"),
    (dict(out=AT[0] + 1024), 4, "overlap q"), (dict(ws=AT[9] + 8, ws_bytes=64), 2, "workspace must be 16B"),
    (dict(max_ctx=1 << 20, ws=AT[0] + 160, ws_bytes=1 << 24), 4, "workspace must not overlap")])
def test_attention_kv8_decode_refusals(lib, kw, code, msg):
    refused(lib, "dk_attention_kv8_decode", DEC, kw, code, msg)


def test_attention_window_workspace(lib):
    need = lib.dk_attention_window_workspace_bytes
    for bad in ((0, 8, 2, 128, 100, 0, 0, 0), (20, 6, 2, 128, 100, 0, 0, 0), (20, 8, 2, 96, 100, 0, 0, 0),
                (20, 8, 2, 128, 0, 0, 0, 0), (20, 8, 2, 128, 100, -1, 0, 0), (20, 8, 2, 128, 100, 0, 0, 3)):
        assert need(*bad) == 0
    big = need(64, 32, 8, 128, 1 << 20, 0, 0, 2)
    assert big % 16 == 0
    if big:                          # a workspace that the call would use must overlap nothing
        kw = dict(M=64, n_q=32, n_kv=8, q_stride=4096, max_ctx=1 << 20, ws_bytes=big)
        for ws in (AT[0] + 160, AT[7] + 16):
            refused(lib, "dk_attention_window", WIN, dict(kw, ws=ws), 4, "workspace must not overlap")


def test_op_module_refusals_on_the_cpu(lib):
    K = ext.DecodeKernels(lib)
    h = lambda *s: torch.zeros(*s, dtype=torch.half)
    bt, pos, f = torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros
    c8, s8 = torch.zeros(4, 2, 16, 64, dtype=torch.int8), f(4, 2, 1)
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.kv8_append_rows(h(3, 384), f(8, 32), f(8, 32), pos, bt, c8, c8, s8, s8, 2, 2)
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.kv8_read(bt, c8, c8, s8, s8, 0, h(3, 2, 64), h(3, 2, 64))
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.attention_window(h(3, 2, 64), pos, bt, h(4, 2, 16, 64), h(4, 2, 16, 64), 10, h(3, 128))
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.attention_kv8(h(3, 2, 64), pos, bt, c8, c8, s8, s8, 10, h(3, 128))
    with pytest.raises(RuntimeError, match="contiguous CUDA tensor"):
        K.attention_kv8_decode(h(384), f(8, 32), f(8, 32), pos, bt, c8, c8, s8, s8, 2, 2, 10, h(128))
    with pytest.raises(RuntimeError, match="int8 or float8_e4m3fn"):
        K.attention_kv8(h(3, 2, 64), pos, bt, h(4, 2, 16, 64), h(4, 2, 16, 64), s8, s8, 10, h(3, 128))
    with pytest.raises(RuntimeError, match="must be fp16"):
        K.attention_window(h(3, 2, 64), pos, bt, c8, c8, 10, h(3, 128))
    with pytest.raises(RuntimeError, match="P / 16"):
        K.attention_kv8(h(3, 2, 64), pos, bt, c8, c8, f(4, 2, 2), s8, 10, h(3, 128))
    with pytest.raises(RuntimeError, match="multiple of 16"):
        K.attention_kv8(h(3, 2, 64), pos, bt, c8[:, :, :8], c8[:, :, :8], s8, s8, 10, h(3, 128))
    with pytest.raises(RuntimeError, match="the cache must be"):
        K.attention_window_workspace_bytes(1, 8, 2, 64, 100, dtype=torch.bfloat16)
    for sizes in ((1, 8, 2, 64, 1 << 32), ((1 << 32) + 1, 8, 2, 64, 100), (1, 8, 2, 64, 100, 1 << 32)):
        with pytest.raises(RuntimeError, match="32 bits"):
            K.attention_window_workspace_bytes(*sizes)


@pytest.mark.parametrize("M,n_q,n_kv,max_ctx", [(64, 32, 8, 1 << 20), (1, 32, 8, 1 << 20), (1, 8, 2, 1 << 14)])
def test_attention_window_workspace_overlaps_nothing(lib, M, n_q, n_kv, max_ctx):
    """Sizes that split, with many columns and with few: the workspace that the call would use is disjoint from q and out."""
    need = lib.dk_attention_window_workspace_bytes(M, n_q, n_kv, 128, max_ctx, 0, 0, 2)
    assert need > 0 and need % 16 == 0
    kw = dict(M=M, n_q=n_q, n_kv=n_kv, q_stride=n_q * 128, max_ctx=max_ctx, ws_bytes=need)
    for ws in (AT[0] + 160, AT[7] + 16, AT[0] - need + 16, AT[7] - need + 16):
        refused(lib, "dk_attention_window", WIN, dict(kw, ws=ws), 4, "workspace must not overlap")
