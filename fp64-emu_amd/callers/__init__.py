"""Callers written against this package: of the emulated GEMM, a left-looking
blocked Cholesky whose updates are batched products (blocked_cholesky.py) and
application drills (drills.py); of the 8-bit operators, a gated MLP trained and
served by all of them together (f8_mlp.py).  Run as scripts for timings at full
size; the GPU tests run them at reduced sizes with accuracy bars."""
