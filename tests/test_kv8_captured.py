"""The calls of the head norms, the 8-bit cache and the controls allocate nothing and can be captured: replays between eager
calls give the eager results, and the device's free memory stays what it was."""
import numpy as np
import pytest

from blog_amd import qlin
from test_kv8 import EPS, _gpu

pytestmark = pytest.mark.gpu


def test_replays_and_memory():
    torch = _gpu()
    from gpu_util import banner
    gen = torch.Generator(device="cuda").manual_seed(4)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    n, heads, kv, d, blocks, rows = 2, 8, 2, 256, 300, 5  # (heads of 256 have registers in scratch)
    table = torch.empty(blocks * 32, d, device="cuda")
    norm = (1 + 0.1 * randn(d)).to(torch.bfloat16)
    qkv = randn(n, rows, (heads + 2 * kv) * d)
    a, width = qkv.data_ptr(), (heads + 2 * kv) * d
    k, v = a + 4 * heads * d, a + 4 * (heads + kv) * d
    cache = qlin.Kv8Cache.empty(torch, n, kv, d, blocks * 32)
    prompt = randn(n, 400, (heads + 2 * kv) * d)
    start, zero, first, lens = i32(400, 27), i32(0, 0), i32(390, 0), i32(405, 32)
    q, q5, q400, attn = randn(n, rows, heads, d), randn(rows, heads, d), randn(n, 400, heads, d), randn(n, rows, heads, d)
    kc, vc = randn(64, kv, d), randn(64, kv, d)
    kr, vr = randn(n, 40, kv, d), randn(n, 40, kv, d)
    logits, picks = randn(3, 50000), i32(0, 0, 0)
    out, history = torch.empty_like(logits), torch.randint(0, 50000, (3, 100), dtype=torch.int32, device="cuda", generator=gen)
    ws = torch.empty(max(qlin.attend_kv8_workspace_bytes(n, rows, heads, kv, d, blocks), qlin.logits_controls_scratch_bytes(3, 50000)),
                     dtype=torch.uint8, device="cuda")
    penalty = torch.full((3,), 0.3, device="cuda")

    qlin.set_stream(torch.cuda.current_stream())
    how = qlin.QkRope(norm, norm, 0, EPS, 0, table, d)
    p = prompt.data_ptr()
    pk, pv = p + 4 * heads * d, p + 4 * (heads + kv) * d
    calls = [
        ("rope_table", lambda: qlin.rope_table(table, 1e5), [table]),
        ("store of a prompt", lambda: qlin.qk_norm_rope_store_kv8(how, cache, p, width, pk, width, pv, width, q400, 400, heads, zero),
         [q400]),
        ("store", lambda: qlin.qk_norm_rope_store_kv8(how, cache, a, width, k, width, v, width, q, rows, heads, start),
         [q, cache.recent, cache.pages]),
        ("f32 store", lambda: qlin.qk_norm_rope_store_kv(how, a, width, k, width, v, width, q5, kc, vc, rows, heads, kv, d, 64,
                                                         first[1:]), [q5, kc, vc]),
        ("read back", lambda: qlin.kv8_read(cache, first, lens, 40, kr, vr), [kr, vr]),
        ("attention", lambda: qlin.attend_kv8(cache, q, attn, rows, heads, start, None, d ** -0.5, ws), [attn]),
        ("controls", lambda: qlin.logits_controls(logits, out, 3, 50000, history=history, frequency=penalty, picks=picks,
                                                  scratch=ws), [out, picks]),
    ]
    # eager, in order; each is repeatable on what the ones before left
    want = []
    for name, call, results in calls:
        banner(name)
        call()
        torch.cuda.synchronize()
        want.append([r.clone() for r in results])
    graphs = []
    for name, call, _ in calls:
        banner(f"capture of {name}")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):  # (an allocation of the library's would end the capture with an error)
            qlin.set_stream(torch.cuda.current_stream())
            call()
        graphs.append(g)
    qlin.set_stream(torch.cuda.current_stream())
    for g in graphs:  # (whatever the runtime allots for a graph's first launch)
        g.replay()
    torch.cuda.synchronize()
    free = lambda: torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved()  # (what torch holds aside)
    for turn in range(4):
        for i in range(len(calls)):
            calls[i][1]()
            graphs[i].replay()
            if turn % 2:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        for (name, _, results), was in zip(calls, want):
            for r, w in zip(results, was):
                assert torch.equal(r, w), (turn, name)
        if turn == 0:  # (the runtime loads code and sets memory aside when it is first asked for)
            before = free()
    assert free() >= before
