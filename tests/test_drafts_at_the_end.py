"""Steps by drafts up to and past the cache's last position: the drafts that have a position are checked, the others are not, and what
is stored and picked is what single steps give."""
import numpy as np
import pytest

from blog_amd import qlin
from test_decoder_kv8 import _close, _env
from test_drafts_rows import _fill, _start
from test_verify_drafts import reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qk_norm,kv8", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("max_seq,n,ahead", [(100, 5, 12), (96, 5, 12), (65, 3, 4), (100, 31, 40), (70, 1, 3), (66, 0, 2)])
def test_up_to_the_last_position(qk_norm, kv8, max_seq, n, ahead):
    torch = _env()
    from gpu_util import banner, host
    banner(f"drafts up to the end: qk_norm={qk_norm} kv8={kv8} max_seq={max_seq} n={n}")
    start = max_seq - ahead
    cfg, dec, twin, d, rng = _start(torch, n, start, qk_norm=qk_norm, kv8=kv8, max_seq=max_seq)
    graph = None
    pos, token, short = start, int(host(dec.token)[0]), 0
    for call in range(40):
        if pos > max_seq + 2:
            break
        at = min(pos, max_seq - 1)
        room = min(n, max_seq - 1 - at)
        short += room < n
        twin.back(at)
        rows, own, drafts = [], token, []
        for i in range(n + 1):
            if i <= room:
                rows.append(twin.run(np.array([own]), at + i)[0])
                own = int(np.argmax(rows[-1])) if rng.random() < 0.7 else int(rng.integers(0, cfg.vocab))
            else:
                own = int(rng.integers(0, cfg.vocab))
            drafts.append(own)
        _fill(torch, d, drafts[:n], n, uniform=0.25)
        d["temperature"].fill_(0.0 if call % 3 else 0.05)
        if call % 2 or graph is None:
            state = dec.token.clone(), dec.pos.clone()
            dec.step_drafts(d)
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                dec.token.copy_(state[0]), dec.pos.copy_(state[1])
                with torch.cuda.graph(graph):
                    dec.step_drafts(d)
                qlin.set_stream(torch.cuda.current_stream())
                dec.token.copy_(state[0]), dec.pos.copy_(state[1])
                graph.replay()
        else:
            graph.replay()
        logits = host(d["logits"])
        for i in range(room + 1):
            assert _close(logits[0, i], rows[i]), (call, pos, i, np.linalg.norm(logits[0, i] - rows[i]) / np.linalg.norm(rows[i]))
        want = reference(logits, np.array([drafts[:n]], np.int32).reshape(1, n), host(d["uniform"]), None, np.array([room], np.int32),
                         host(d["temperature"]))
        m = int(want[1][0])
        assert np.array_equal(host(d["tokens"]), want[0]) and int(host(d["accepted"])[0]) == m and m <= room
        assert (host(d["rates"])[0, room:] == 0).all() and int(host(d["n_drafts"])[0]) == n
        pos, token = pos + m + 1, int(want[0][0, m])
        assert int(host(dec.pos)[0]) == pos and int(host(dec.token)[0]) == token
        twin.back(min(pos, max_seq))
    assert pos > max_seq + 2 and (short > 2 or n == 0)
    at = max_seq - 1
    twin.back(at)
    want = twin.run(np.array([token]), at)[0]
    dec.step()
    assert _close(host(dec.logits), want)
