"""HIP kernels behind nlearn's ``nlearn.kernels`` entry points (gemm, cross_entropy), and beside them fp8 and distill."""
