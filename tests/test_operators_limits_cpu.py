"""More refusals of the device operators (no GPU needed): counts at the ends of their ranges."""
import pytest

from tests.test_operators_cpu import conv, scan

REFUSED = [
    (lambda: conv(n_seq=(1 << 31) - 1), "n_seq must be"), (lambda: conv("rec_history_conv_backward", n_seq=(1 << 31) - 1), "n_seq must be"),
    (lambda: scan(n_seq=(1 << 31) - 1), "n_seq must be"), (lambda: scan("rec_history_scan_step", n_seq=(1 << 31) - 1), "n_seq must be"),
    (lambda: conv(n_seq=(1 << 31) - 2, device=99), "no such HIP device"), (lambda: scan(n_seq=(1 << 31) - 2, device=99), "no such HIP device"),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refused_with_a_reason(case):
    f, words = REFUSED[case]
    rc, said = f()
    assert rc == -1 and words in said, (rc, said)
