"""Sizes that between them run every compiled kernel of the fused products, with every number of parts that a
tile's reduction is cut into (test_fused_choice.py holds the list to that)."""

# tokens, d_model, d_ff
BLOCK = [
    (1, 16, 19), (1, 2292, 9708), (1, 1590, 2901), (1646, 20, 1420), (1, 2299, 2065), (1, 8850, 4953), (1931, 18, 1034),
    (1, 4780, 13757), (1325, 20, 18), (1, 2178, 867), (1, 1021, 3438), (4870, 4488, 16), (1, 2127, 20779),
    (148, 4920, 456), (12810, 16, 756), (4434, 663, 164), (146, 1604, 4798), (129, 4968, 2128), (159, 2477, 4957),
    (412, 4891, 648), (16049, 141, 644), (175, 1232, 8992), (11370, 130, 1586), (134, 2458, 8018), (406, 4882, 1416),
    (148, 5452, 5467), (143, 8972, 4070), (129, 2767, 15428), (261, 4927, 11023), (1943, 936, 8656)]
# matrices, rows, columns
UPDATE = [
    (1, 17, 16), (1, 16, 19), (5, 3655, 18), (2, 130, 5164), (8, 1653, 129), (16, 17, 1475), (16, 131, 1764),
    (16, 1579, 129), (16, 1172, 385), (16, 399, 1221), (3, 1201, 1426), (1, 900, 4776), (1, 4930, 897), (2, 1722, 1422),
    (8, 1325, 1288), (16, 529, 2476), (3, 777, 10125), (5, 8939, 679)]

# numbers of csrc/fused_gemm.h: FusedOp, and the operand types
GATE, DOWN, DACT, DX, DW, GRAM_WIDE, GRAM_TALL, POLY, UPDATE_WIDE, UPDATE_TALL = range(10)
BF16, F16 = 1, 2


def block_products(tokens, d, f, dt):
    """The products of a forward and a backward call: (op, type, M, N, K, matrices)."""
    return [(GATE, dt, tokens, f, d, 1), (DOWN, dt, tokens, d, f, 1), (DACT, dt, tokens, f, d, 1),
            (DX, dt, tokens, d, f, 1), (DW, dt, f, d, tokens, 2)]


def update_products(batch, rows, cols):
    """The products of a step of an orthogonalisation."""
    m, n, tall = min(rows, cols), max(rows, cols), rows > cols
    return [(GRAM_TALL if tall else GRAM_WIDE, F16, m, m, n, batch), (POLY, F16, m, m, m, batch),
            (UPDATE_TALL if tall else UPDATE_WIDE, F16, rows, cols, m, batch)]
