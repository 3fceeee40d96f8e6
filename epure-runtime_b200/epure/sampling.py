"""Which drafted tokens a target model keeps (include/epq_sampling.h).

The reference generates through the Hugging Face model, one token a pass.  A draft (a smaller model, or text looked up in
what was generated so far) lets a pass of the target judge several tokens at once: ``verify`` accepts as many of them as
leaves the output distributed as the target's own, and draws the token behind them, from random numbers that it is given.
"""
from . import _native


def verify(target, draft, tokens, uniforms):
    """Verification of drafted tokens by rejection: ``(tokens [batch, drafts + 1], accepted [batch])``, both int64.

    ``target`` [batch, drafts + 1, vocab] holds the target's probabilities p for the place of each drafted token and the one
    behind them, ``draft`` [batch, drafts, vocab] (of the same type) those q that the tokens were drawn with, or None for
    tokens without any (looked up, or greedy: each counts as certain).  ``tokens`` (int64 [batch, drafts]) are the drafts, a
    row's ending at its first negative one; ``uniforms`` (float32 [batch, drafts + 1]) random numbers of [0, 1).

    Draft i is accepted while ``u_i q_i(x_i) < p_i(x_i)``.  Behind the accepted ones one token is drawn with the row's last
    number: at a refused draft from ``max(p - q, 0)`` (without a draft's probabilities: p without the token), else from p.
    The result holds a row's accepted drafts, the drawn token, and -1 behind it.  Products are 64-bit and sums keep 45 bits or more, so
    the drawn token is the definition's (but where the number lies that near a token's edge); without drafts (``tokens`` [batch, 0]) this samples from the target."""
    return (_native.tensor_calls or _native.load_tensor_calls()).verify(target, draft, tokens, uniforms)
