"""MI355X-native exact Gaussian-process regression hot path behind the reference's Python API
(emakryo/gaussian_process: kernels.py, regression.py, expectation_propagation.py, distillation.py)."""
from .regression import GaussianProcessRegression
from .expectation_propagation import GaussianProcessExpectationPropagation
from .distillation import GaussianProcessDistillation
from .kernels import RBF, ARD, KernelValue
from .delta import gated_delta_rule, gated_delta_rule_backward, gated_delta_rule_step
from .orthogonal import orthogonalize

__all__ = ["GaussianProcessRegression", "GaussianProcessExpectationPropagation",
           "GaussianProcessDistillation", "RBF", "ARD",
           "KernelValue", "gated_delta_rule", "gated_delta_rule_backward", "gated_delta_rule_step",
           "orthogonalize"]
