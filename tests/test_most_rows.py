"""More rows than one launch holds (2^32 threads) are refused as a limit, before anything is launched."""
import pytest

from blog_amd import qlin

OK, UNSUP, SHAPE, NULL, ROWB, LIMIT, LAUNCH, ALIGN = range(8)
FAKE = 0x10000


@pytest.mark.parametrize("rows,hidden", [(2 ** 31 - 1, 1), (2 ** 31 - 1, 256), (1 << 26, 256), (1 << 24, 1024), (1 << 24, 4096), (1 << 23, 2048 * 2 + 1), (1 << 22, 20000)])
def test_add_rms_norm(rows, hidden):
    assert qlin.status("qlin_launch_add_rms_norm", FAKE, hidden, 0, 0, 0, 0, FAKE, 0, 1e-6, 0, FAKE, hidden, 0, 0, 0, rows, hidden) == LIMIT


@pytest.mark.parametrize("tokens,experts", [(2 ** 31 - 1, 8), (1 << 26, 8), ((1 << 26) + 5, 1024)])
def test_moe_route(tokens, experts):
    how = qlin.MoeRouting()
    assert qlin.status("qlin_launch_moe_route", how.address, FAKE, experts, FAKE, FAKE, tokens, experts, 2) == LIMIT


def test_verify_drafts():
    n, vocab = 1 << 22, 100
    need = qlin.verify_drafts_workspace_bytes(n, 0, vocab)
    assert qlin.status("qlin_launch_verify_drafts", FAKE, vocab, 0, 0, 0, 0, 0, FAKE, FAKE, FAKE, 0, 0, n, 0, vocab, FAKE, need) == LIMIT
