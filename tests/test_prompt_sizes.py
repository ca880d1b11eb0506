"""Sizes that prompt_attention takes, prompt_attention_bwd takes too: a training program would find out
behind its forward.  Without a GPU: the workspaces' sizes tell (-1: refused)."""
import pytest

LIMIT = 1 << 24                                            # workgroups


def sizes(lib, *a):
    return (lib.fagq_prompt_attention_workspace_bytes(*a), lib.fagq_prompt_attention_bwd_workspace_bytes(*a))


def slots(T, B):
    """Tiles of 128 rows that T rows of B sequences may need."""
    return (T + B * 127 + 127) // 128


@pytest.mark.parametrize("B,T,Hq,H,D", [
    (65536, 524288, 16, 16, 128), (32768, 524288, 32, 32, 128), (1, 1 << 20, 128, 128, 64), (1, 1 << 20, 64, 64, 128),
    (2100, 2300, 4096, 4096, 64), (1, 1 << 24, 96, 96, 256), (1, 1 << 24, 96, 8, 256), (1 << 20, 1 << 20, 8, 8, 128),
    (1 << 23, 16000, 1, 1, 64), (1 << 23, 16000, 1, 1, 256), (1 << 22, 100, 2, 2, 128), (1 << 23, 0, 1, 1, 64),
])
def test_the_backward_takes_what_the_forward_takes(lib, B, T, Hq, H, D):
    f, b = sizes(lib, B, T, T, Hq, H, D)
    assert f >= 0 and b >= 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,Hq,H", [(B, Hq, H) for B in (1, 7, 1000, 1 << 20)
                                    for Hq, H in ((1, 1), (8, 8), (64, 64), (64, 8), (4096, 4096)) if B * Hq < LIMIT])
def test_up_to_the_limit(lib, B, Hq, H, D):
    """The last number of tokens below 2^24 workgroups, and the first above."""
    T = LIMIT // Hq * 128 - B * 127 - 127
    for rows in (T - 129, T - 128, T - 1, T, T + 128):
        if not 0 <= rows < (1 << 31) - 1024:
            continue
        f, b = sizes(lib, B, rows, rows, Hq, H, D)
        assert (f >= 0) == (b >= 0) == (slots(rows, B) * Hq < LIMIT), rows


def test_keys_past_the_limit(lib):
    """Few queries over more tiles of keys than a grid holds: the gradients' own limit."""
    few = lambda Tk, H: sizes(lib, 1, 128, Tk, 64, H, 64)
    assert min(few(1 << 24, 64)) >= 0
    f, b = few(1 << 25, 64)
    assert f >= 0 and b == -1
