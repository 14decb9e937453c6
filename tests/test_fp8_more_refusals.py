"""Arguments of the 8-bit row and routing calls that were cut or written over one another, refused before anything is launched."""
from tests.test_fp8_refusals_cpu import A, B, S, bind


def quantise(fake, rows, K, sr, sb):
    fake.fake_reset(0)
    ld = (K + 15) // 16 * 16
    return fake.coli_b200_quantize_rows_fp8(0, A, 2, K, None, rows, rows, K, B, ld, S, sr, sb, None), fake.fake_queued()


def test_columns(fake_cuda):
    fake, most = bind(fake_cuda), 65535 * 1024
    assert quantise(fake, 1, most, 0, 1) == (1, 1)
    for K in (most + 1, 2**31 - 1100, 2**31 - 300, 2**31 - 256, 2**31 - 1):  # (the grid's columns of these pass 32 bits)
        assert quantise(fake, 1, K, 0, 1) == (0, 0), K


def test_scales_in_one_place(fake_cuda):
    fake = bind(fake_cuda)
    for rows, K, sr, sb in ((5, 300, 1, 5), (5, 300, 3, 1), (5, 300, 7, 2), (5, 300, 2, 3), (1, 300, 0, 1), (5, 100, 1, 0), (1, 128, 0, 0), (5, 300, 3, 15), (5, 300, 9, 6)):
        places = {r * sr + b * sb for r in range(rows) for b in range((K + 127) // 128)}
        fits = len(places) == rows * ((K + 127) // 128)
        assert quantise(fake, rows, K, sr, sb) == ((1, 1) if fits else (0, 0)), (rows, K, sr, sb)
    for rows, K, sr, sb in ((5, 300, 0, 1), (5, 300, 1, 0), (5, 300, 0, 0), (5, 300, 1, 1), (5, 300, 1, 4), (2, 300, 1, 1), (5, 128, 0, 1)):
        assert quantise(fake, rows, K, sr, sb) == (0, 0), (rows, K, sr, sb)
