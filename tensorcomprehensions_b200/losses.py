"""Losses of a large-vocabulary head with torch.autograd support, next to the layers that comprehensions build.

    loss = tc.linear_cross_entropy(X, W, target)                  # [N]; no [N, V] logits are kept
    (loss.sum() / (target != -100).sum()).backward()              # dX, dW

    logits = T.matmul(X, W)                                       # any student logits [N, V]
    loss = tc.topk_distillation(logits, indices, teacher, temperature=2.0)

Both run on tensors of one CUDA device, on its current stream, without synchronising; they may be captured into CUDA graphs (a
backward pass while no eager graph of the same leaves lives: torch's autograd would wait for that graph's stream, and raises).
There is no CPU or eager fallback, no second derivative and no forward-mode one: a dual tensor raises.  The reference's operator library has no loss (its tc/library ends at the layers).
"""
from . import tclib


def linear_cross_entropy(X, W, target, ignore_index=-100):
    """Softmax cross entropy of the linear layer z = X W^T, one float32 value a row, without keeping z:

        loss[n] = log(sum_v exp z[n, v]) - z[n, target[n]]

    X [N, D] and W [V, D]: float32, float16 or bfloat16, of one type, dense along D, rows any distance apart.  target [N]:
    int32 or int64.  A row with target == ignore_index has loss 0 and gradient 0, and what its X holds does not matter; a
    target outside [0, V) makes the row's loss NaN, and with it the gradients of that row of X and of W.  Gradients of
    X and W have their type, are summed in float32 and rounded once.  Between the two products the gradient of z is rounded to
    the inputs' 16-bit type, relative to the batch's largest gradient of a loss (float16: rows below 2^-16 of it have a scale of
    their own in X's gradient; W's loses what lies below 2^-39 of it).  float32 products take operands of 22 significand bits for
    the logits, relative to a row of X or W down to 2^-29 of its largest value, and of 24 for the gradients: float32 accuracy.
    If a wait inside a kernel gives up (never on a sound device), the loss, or both gradients, are NaN.  A wrong type, size, stride or device
    raises RuntimeError."""
    return tclib.linear_cross_entropy(X, W, target, ignore_index)


def topk_distillation(logits, indices, teacher, temperature=1.0):
    """Kullback-Leibler divergence of a student's distribution from a teacher's K largest logits, one float32 value a row:

        q = softmax(teacher / T) over the row's entries,  p = softmax(logits / T) over V
        loss[n] = T^2 sum_k q[k] (ln q[k] - ln p[indices[n, k]])

    logits [N, V] and teacher [N, K]: float32, float16 or bfloat16; indices [N, K]: int32 or int64; all dense along their
    last dimension; 1 <= K <= 4096; T > 0, its square a normal float32 number (2^-63 <= T < 2^64).  An index below 0, or a teacher logit of -inf, is no entry; a row without entries has
    loss 0 and gradient 0; an index of V or more makes the row's loss and gradient NaN; an index that stands twice counts
    twice.  The gradient is that of the logits, in their type; the teacher gets none.  A wrong type, size, stride,
    device or temperature raises RuntimeError."""
    return tclib.topk_distillation(logits, indices, teacher, temperature)
